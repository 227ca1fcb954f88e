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
// A warp takes one (sequence, kv head, split of the history) by itself: the records of its blocks stream
// through a ring of its own in shared memory, one bulk copy a block, and nothing but that ring's barriers
// is waited for. The running maximum moves only when a score passes it by 2^6 (a vote per 16 keys; the
// first ones set it), so most runs shuffle nothing. A second kernel joins the splits. How a history is
// cut depends on its length alone: a sequence's result does not depend on the batch.
#include <algorithm>
#include <atomic>

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

// Keys of a split: short where a lone sequence needs the warps, longer where the ends of a split (query
// in, partial result out) would cost more than they bring. At most 32 blocks, whose table entries a warp
// holds one a lane.
__host__ __device__ __forceinline__ int part_of(int n) { return n <= 1024 ? 128 : n <= 4096 ? 256 : 512; }
// Splits of a history of n keys.
__host__ __device__ __forceinline__ int splits_of(int n) { return n <= 128 ? 1 : (n + part_of(n) - 1) / part_of(n); }

template <int D, int NG, int BS>
struct Ring {
  // stages of a record each: 9 KB and more a warp, so that four CTAs of an SM keep over 100 KB on the way
  static constexpr int kStages = Rec<D, NG, BS>::kBytes > 4096 ? 3 : 9216 / Rec<D, NG, BS>::kBytes;
  static constexpr int kBytes = kStages * Rec<D, NG, BS>::kBytes;
  static constexpr int kSmem = kDecWarps * (kBytes + 8 * kStages);
};

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

// Key (of 16) that row r of S^T stands for: rows 2 i and 2 i + 1, whose keys a lane's P and V pair up, are
// keys i and (i ^ 1) + 4, so that the eight lanes of a 16-byte shared load meet both halves of the banks.
ES_DEVICE int key_of_row(int r) { return (r & 8) + ((r & 1) ? ((r >> 1 & 3) ^ 1) + 4 : (r >> 1 & 3)); }

// What a lane (gid = lane / 4, tig = lane % 4) holds of a run of 16 keys.
template <int D, int NG>
struct Run {
  uint32_t k[2][D / 32];          // K words of rows gid and gid + 8
  uint32_t v[4][D / 64];          // V words of rows 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
  uint32_t kp[2][NG], vp[2][NG];  // (scale, zero) pairs of rows gid and gid + 8
};

template <int D, int NG, int BS>
ES_DEVICE void load_run(Run<D, NG>& r, const uint8_t* rec, int sub, int gid, int tig) {
  using R = Rec<D, NG, BS>;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int row = sub * 16 + 8 * i + key_of_row(gid);
    const uint8_t* kp = rec + row * R::kRow + tig * (D / 8);
    if (D == 128) {
      const uint4 w = *reinterpret_cast<const uint4*>(kp);
      r.k[i][0] = w.x, r.k[i][1] = w.y, r.k[i][D / 32 - 2] = w.z, r.k[i][D / 32 - 1] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(kp);
      r.k[i][0] = w.x, r.k[i][1] = w.y;
    }
    const uint8_t* mp = rec + R::kKMeta + row * R::kMeta;
    if (NG == 2) {
      const uint2 a = *reinterpret_cast<const uint2*>(mp);
      const uint2 b = *reinterpret_cast<const uint2*>(mp + BS * R::kMeta);
      r.kp[i][0] = a.x, r.kp[i][NG - 1] = a.y, r.vp[i][0] = b.x, r.vp[i][NG - 1] = b.y;
    } else {
      r.kp[i][0] = *reinterpret_cast<const uint32_t*>(mp);
      r.vp[i][0] = *reinterpret_cast<const uint32_t*>(mp + BS * R::kMeta);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int row = sub * 16 + 8 * (j >> 1) + ((j & 1) ? (tig ^ 1) + 4 : tig);
    const uint8_t* vp = rec + R::kV + row * R::kRow + gid * (D / 16);
    if (D == 128) {
      const uint2 w = *reinterpret_cast<const uint2*>(vp);
      r.v[j][0] = w.x, r.v[j][D / 64 - 1] = w.y;
    } else {
      r.v[j][0] = *reinterpret_cast<const uint32_t*>(vp);
    }
  }
}

// The running state of a warp's 8 query heads over its keys.
template <int D, int NG>
struct Acc {
  float o[D / 16][4];       // O^T tiles of the codes: (channel gid | gid + 8 of the tile, heads 2 tig, 2 tig + 1)
  float m[2], l[2];         // of heads 2 tig and 2 tig + 1; l and zs: this lane's keys alone
  float zs[2][NG];          // sum P * zero
  int ve;                   // V scales enter f16 times vf = 2^(kPBits - ve)
  float vf, vlim;           // and are at most vlim
};

// One run of 16 keys; kTail: only the first `valid` of them count, and whatever the other slots hold (NaN
// too) is taken out of the products.
template <int D, int NG, bool kTail>
ES_DEVICE void attend(Acc<D, NG>& A, const Run<D, NG>& r, const uint32_t (*qb)[4], const float* xs, const float (*sq)[NG],
                      int gid, int valid) {
  constexpr int KW = D / 32, VW = D / 64, MT = D / 16;
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
  // scores in the log2 domain: x[row i][head j]
  float x[2][2], sv[2][NG], zv[2][NG];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const bool in = !kTail || key_of_row(gid) + 8 * i < valid;
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
  const bool up = fmaxf(x[0][0], x[1][0]) > A.m[0] + kSlack || fmaxf(x[0][1], x[1][1]) > A.m[1] + kSlack || smax > A.vlim;
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
      const float mn = fmaxf(A.m[j], mt[j]);
      c[j] = A.m[j] == -INFINITY ? 0.f : ex2(A.m[j] - mn);
      A.m[j] = mn;
      A.l[j] *= c[j];
#pragma unroll
      for (int g = 0; g < NG; g++) A.zs[j][g] *= c[j];
    }
    if (smax > A.vlim) {
      const int e = exponent(smax) + 1;
      const float f = pow2i(max(-126, A.ve - e));
      c[0] *= f, c[1] *= f;
      A.ve = e;
      A.vf = pow2i((int)kPBits - e);
      A.vlim = pow2i(e + 2);
    }
#pragma unroll
    for (int i = 0; i < MT; i++) A.o[i][0] *= c[0], A.o[i][1] *= c[1], A.o[i][2] *= c[0], A.o[i][3] *= c[1];
  }
  // P, its sums, and P * scale as the B fragments of O^T (keys along k): transposed in registers
  float pr[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      pr[i][j] = ex2(x[i][j] - A.m[j]);
      A.l[j] += pr[i][j];
#pragma unroll
      for (int g = 0; g < NG; g++) A.zs[j][g] = fmaf(pr[i][j], zv[i][g], A.zs[j][g]);
    }
  uint32_t pb[NG][2];
#pragma unroll
  for (int g = 0; g < NG; g++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float s = sv[i][g] * A.vf;
      pb[g][i] = transpose8(pack_f16x2(pr[i][0] * s, pr[i][1] * s));
    }
  // O^T += V^T . P^T on the codes: rows gid and gid + 8 of tile (w, j) are channels 2 j and 2 j + 1 of
  // word w, a register's halves the keys of rows 2 tig and 2 tig + 1
#pragma unroll
  for (int w = 0; w < VW; w++) {
    const int g = NG == 2 ? w : 0;
    uint32_t e0 = __byte_perm(r.v[0][w], r.v[1][w], 0x5410), d0 = __byte_perm(r.v[0][w], r.v[1][w], 0x7632);
    uint32_t e1 = __byte_perm(r.v[2][w], r.v[3][w], 0x5410), d1 = __byte_perm(r.v[2][w], r.v[3][w], 0x7632);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t a0[4] = {e0 & 0x000F000Fu, d0 & 0x000F000Fu, e1 & 0x000F000Fu, d1 & 0x000F000Fu};
      mma_f16_16816(A.o[w * 4 + 2 * h], a0, pb[g][0], pb[g][1]);
      const uint32_t a1[4] = {e0 & 0x00F000F0u, d0 & 0x00F000F0u, e1 & 0x00F000F0u, d1 & 0x00F000F0u};
      mma_f16_16816(A.o[w * 4 + 2 * h + 1], a1, pb[g][0], pb[g][1]);
      e0 >>= 8, d0 >>= 8, e1 >>= 8, d1 >>= 8;
    }
  }
}

template <int D, int NG, int BS>
__global__ void __launch_bounds__(kDecThreads, 4) decode_kernel(DecodeParams p) {
  using R = Rec<D, NG, BS>;
  using C = Ring<D, NG, BS>;
  constexpr int KW = D / 32;  // K words a lane holds of a key
  constexpr int VW = D / 64;  // V words
  constexpr int ST = C::kStages;
  extern __shared__ __align__(128) uint8_t smem[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x * kDecWarps + warp, b = blockIdx.z;
  const int kvh = blockIdx.y / p.head_tiles, ht = blockIdx.y % p.head_tiles;
  const int G = p.hq / p.hkv;
  const int heads = min(8, G - ht * 8);  // query heads of this tile
  const int head0 = kvh * G + ht * 8;
  const int gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = smem + warp * C::kBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kDecWarps * C::kBytes) + warp * ST;
  if (lane == 0) {
    for (int i = 0; i < ST; i++) ptx::mbar_init(&full[i], 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();

  pdl_wait();
  pdl_launch();
  const int ctx = min(p.ctx_lens[b], p.bt_cols * BS);
  if (ctx <= 0) {
    if (split == 0)  // an empty history: the output is zero
      for (int i = lane; i < heads * D; i += 32) p.out[((int64_t)b * p.hq + head0) * D + i] = f2bf(0.f);
    return;
  }
  const int ns = min(p.max_splits, splits_of(ctx));
  const int plen = ((ctx + ns - 1) / ns + BS - 1) / BS * BS;  // equal splits, to a block
  const int s0 = split * plen, s1 = min(ctx, s0 + plen);
  if (split >= ns) return;
  const int64_t row0 = (int64_t)b * p.hq + head0;
  const int blocks = (s1 - s0 + BS - 1) / BS;

  // the block table's entries, 32 at a time, one a lane
  const int* bt = p.block_tables + (int64_t)b * p.bt_stride + s0 / BS;
  auto entries = [&](int first) {
    int64_t blk = first + lane < blocks ? bt[first + lane] : 0;
    if (blk < 0 || blk >= p.num_blocks) {  // not a block of this cache: reported, block 0 read instead
      if (p.status) atomicExch(p.status, (int)kBadShape);
      blk = 0;
    }
    return (int)blk;
  };
  int ids = entries(0);
  const uint8_t* head_base = p.cache + (int64_t)kvh * R::kBytes;
  const uint64_t pol = ptx::policy_evict_first();
  auto issue = [&](int i) {
    const int64_t blk = __shfl_sync(0xffffffffu, ids, i & 31);
    if (lane == 0) {
      ptx::mbar_arrive_expect_tx(&full[i % ST], R::kBytes);
      ptx::bulk_g2s_hint(ring + i % ST * R::kBytes, head_base + blk * p.s_block, R::kBytes, &full[i % ST], pol);
    }
  };
  int issued = min(ST, blocks);
  for (int i = 0; i < issued; i++) issue(i);

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

  Acc<D, NG> A;
#pragma unroll
  for (int i = 0; i < D / 16; i++) A.o[i][0] = A.o[i][1] = A.o[i][2] = A.o[i][3] = 0.f;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    A.m[j] = -INFINITY, A.l[j] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; g++) A.zs[j][g] = 0.f;
  }
  A.ve = -90;
  A.vf = pow2i((int)kPBits + 90);
  A.vlim = 0.f;

  for (int i = 0; i < blocks; i++) {
    const uint8_t* rec = ring + i % ST * R::kBytes;
    if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[i % ST], (i / ST) & 1))) {
      // the copies on their way have to land before the warp leaves
      for (int k = i; k < issued; k++) ptx::mbar_wait(&full[k % ST], (k / ST) & 1);
      if (lane == 0 && p.status) atomicExch(p.status, (int)kTimeout);
      return;
    }
#pragma unroll
    for (int sub = 0; sub < BS / 16; sub++) {
      const int valid = s1 - s0 - i * BS - sub * 16;
      if (valid <= 0) break;
      Run<D, NG> r;
      load_run<D, NG, BS>(r, rec, sub, gid, tig);
      if (sub == BS / 16 - 1 && issued < blocks) {
        __syncwarp();  // every lane has read the stage
        if ((issued & 31) == 0) ids = entries(issued);
        issue(issued++);
      }
      if (valid >= 16)
        attend<D, NG, false>(A, r, qb, xs, sq, gid, 16);
      else
        attend<D, NG, true>(A, r, qb, xs, sq, gid, valid);
    }
  }

  // the lanes' sums; the output with the codes' factor and the zeros' part
#pragma unroll
  for (int s = 4; s < 32; s <<= 1) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      A.l[j] += __shfl_xor_sync(0xffffffffu, A.l[j], s);
#pragma unroll
      for (int g = 0; g < NG; g++) A.zs[j][g] += __shfl_xor_sync(0xffffffffu, A.zs[j][g], s);
    }
  }
  const float of = pow2i(24 - (int)kPBits + A.ve);
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int h = 2 * tig + j;
    if (h >= heads) continue;
    const float inv = 1.f / A.l[j];
#pragma unroll
    for (int w = 0; w < VW; w++) {
      float y[8];  // channels 8 (gid + 8 w) and up
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float f = (i & 1) ? of * 0.0625f : of, z = A.zs[j][NG == 2 ? w : 0];
        y[2 * i] = fmaf(A.o[w * 4 + i][j], f, z);
        y[2 * i + 1] = fmaf(A.o[w * 4 + i][2 + j], f, z);
      }
      const int ch = 8 * (gid + 8 * w);
      if (ns == 1) {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] *= inv;
        *reinterpret_cast<uint4*>(p.out + (row0 + h) * D + ch) = pack8(y);
      } else {
        float4* po = reinterpret_cast<float4*>(p.part_o + ((row0 + h) * p.max_splits + split) * D + ch);
        po[0] = make_float4(y[0], y[1], y[2], y[3]);
        po[1] = make_float4(y[4], y[5], y[6], y[7]);
      }
    }
    if (ns > 1 && gid == 0)
      *reinterpret_cast<float2*>(p.part_ml + ((row0 + h) * p.max_splits + split) * 2) = make_float2(A.m[j], A.l[j]);
  }
}

// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a row's splits, in an order of its own: warp w
// takes splits w, w + 8, ..., then the warps add in order. One CTA per (sequence, query head); the loads of
// four splits are on the way at a time.
constexpr int kMergeWarps = 8;
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32)
    merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ ctx_lens,
                 __nv_bfloat16* __restrict__ out, int hq, int max_splits, int max_keys) {
  constexpr int E = D / 32;  // neighbouring channels of a lane
  __shared__ float so[kMergeWarps][D], sl[kMergeWarps], smx[kMergeWarps];
  pdl_wait();
  pdl_launch();
  const int ns = min(max_splits, splits_of(min(ctx_lens[blockIdx.y], max_keys)));
  if (ns <= 1) return;  // written by the split itself
  const int64_t row = (int64_t)blockIdx.y * hq + blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + row * max_splits;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < ns; i += kMergeWarps * 32) mx = fmaxf(mx, ml[i].x);
  mx = warp_max(mx);
  if (lane == 0) smx[warp] = mx;
  __syncthreads();
  mx = smx[0];
#pragma unroll
  for (int w = 1; w < kMergeWarps; w++) mx = fmaxf(mx, smx[w]);
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.f;
  const float* po = part_o + row * max_splits * D + E * lane;
#pragma unroll 4
  for (int i = warp; i < ns; i += kMergeWarps) {
    const float2 t = ml[i];
    const float f = t.x == mx ? 1.f : ex2(t.x - mx);
    l = fmaf(t.y, f, l);
    float v[E];
    if (E == 4) {
      const float4 x = *reinterpret_cast<const float4*>(po + (int64_t)i * D);
      v[0] = x.x, v[1] = x.y, v[E - 2] = x.z, v[E - 1] = x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(po + (int64_t)i * D);
      v[0] = x.x, v[1] = x.y;
    }
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = fmaf(v[e], f, acc[e]);
  }
#pragma unroll
  for (int e = 0; e < E; e++) so[warp][E * lane + e] = acc[e];
  if (lane == 0) sl[warp] = l;
  __syncthreads();
  if (threadIdx.x < D) {
    const int c = threadIdx.x;
    float t = so[0][c], lt = sl[0];
#pragma unroll
    for (int w = 1; w < kMergeWarps; w++) t += so[w][c], lt += sl[w];
    out[row * D + c] = f2bf(t / lt);
  }
}

template <int D, int NG, int BS>
cudaError_t launch_decode(const DecodeParams& p, int B, cudaStream_t stream) {
  using C = Ring<D, NG, BS>;
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = once_per_device(configured, [] {
    return cudaFuncSetAttribute(decode_kernel<D, NG, BS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return e;
  e = launch_ex(decode_kernel<D, NG, BS>, dim3((p.max_splits + kDecWarps - 1) / kDecWarps, p.hkv * p.head_tiles, B),
                dim3(kDecThreads), C::kSmem, stream, 0, p);
  if (e != cudaSuccess || p.max_splits == 1) return e;
  return launch_ex(merge_kernel<D>, dim3(p.hq, B), dim3(kMergeWarps * 32), 0, stream, 0, (const float*)p.part_o,
                   (const float*)p.part_ml, p.ctx_lens, p.out, p.hq, p.max_splits, p.bt_cols * BS);
}

}  // namespace kv4

int64_t kv4_max_splits(int64_t max_len) {
  // the most of any length up to max_len: the count falls where the splits get longer
  const int n = (int)std::min<int64_t>(max_len, INT32_MAX - 1024);
  int most = kv4::splits_of(n);
  for (const int top : {1024, 4096})
    if (n > top) most = std::max(most, kv4::splits_of(top));
  return most;
}

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
