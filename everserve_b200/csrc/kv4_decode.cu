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
// of two, which keeps its bf16 values exact in f16 down to 2^-24. The zeros' part of the scores is one
// m16n8k8 on the bf16 zeros as stored, against sum q split into three bf16 terms (24 bits). P_t scale_tg
// is rounded to f16 (11 bits) under a power of two that follows the largest scale seen; scores, sums, the
// zeros' part and the output stay in fp32.
//
// A warp takes one (sequence, kv head, split of the history) by itself: the records of its blocks stream
// through a ring of its own in shared memory, one bulk copy a block, and nothing but that ring's barriers
// is waited for. The running maximum moves only when a score passes it by 2^6 (a vote per 32 keys; the
// first ones set it), so most steps shuffle nothing. The splits of a pair are neighbouring warps: where a CTA
// holds all of them (histories up to 2048 keys) it joins them itself, else a second kernel does, in the same
// order. How a history is cut depends on its length alone: a sequence's result does not depend on the batch.
//
// Measured: 2 sequences of 126K keys (32 / 8 heads of 128, 289 MB) in 69 us, 4.2 of the copy's 6.5 TB/s; 48 of
// up to 8K (64 / 8 heads) in 58 us; 64 of 1K in 27 us. Bound by latency and issue: 280 instructions for 16 keys of a
// kv head, 88 of them masks, shifts and permutes on the integer pipe, at 2.3 of 4 a cycle with 16 warps an SM
// (20 warps spill: 82 us for the first).
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
constexpr int kDecCtas = 4;  // a SM (8 warps and 2 CTAs: 62 us against 56 for 48 ragged sequences)
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kSlack = 6.f;       // log2 of how far a score may pass the running maximum
constexpr int kPBits = 7;           // P * scale enters f16 as at most 2^(6 + 2 + 7) = 2^15

// Keys of a split: short where a lone sequence needs the warps, longer where the ends of a split (query
// in, partial result out) cost more than they bring (64 sequences of 1K keys: 29.5 us at 256, 32.2 at 128;
// 48 of up to 8K: 57.0 at 512, 58.1 at 256).
__host__ __device__ __forceinline__ int part_of(int n) { return n <= 1024 ? 256 : 512; }
// Splits of a history of n keys.
__host__ __device__ __forceinline__ int splits_of(int n) { return n <= 256 ? 1 : (n + part_of(n) - 1) / part_of(n); }

template <int D, int NG, int BS>
struct Ring {
  // stages of a record each, about 14 KB a warp (an even count, as a step of 32 keys may take two)
  static constexpr int kStages = Rec<D, NG, BS>::kBytes > 4096 ? 3 : 13824 / Rec<D, NG, BS>::kBytes / 2 * 2;
  static constexpr int kBytes = kStages * Rec<D, NG, BS>::kBytes;
  static constexpr int kStep = 32 / BS;                 // blocks of a step of 32 keys, which share a barrier
  static constexpr int kSteps = kStages / kStep;
  static constexpr int kSmem = kDecWarps * (kBytes + 8 * kSteps);
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
  int join;  // a pair's splits are one CTA's, which joins them
  float scale_log2;
};

ES_DEVICE void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D (16x8 fp32) = A (16x8 bf16, row) * B (8x8 bf16, col) + C, C the same in every row
ES_DEVICE void mma_bf16_1688(float* d, uint32_t a0, uint32_t a1, uint32_t b, float c0, float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%7,%8};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b), "f"(c0), "f"(c1));
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

// The running state of a warp's 8 query heads over its keys. With k = kPBits - ve, probabilities are kept
// as 2^(score - m + k), so that times a V scale (at most 2^(ve + 2)) they fit f16.
template <int D, int NG>
struct Acc {
  float o[D / 16][4];  // O^T tiles of the codes: (channel gid | gid + 8 of the tile, heads 2 tig, 2 tig + 1)
  float m[2], l[2];    // of heads 2 tig and 2 tig + 1; l and zs: this lane's keys alone
  float zs[2][NG];     // sum P * zero
  float k, vlim;       // the exponent above, and the scales it holds for
};

// What a warp keeps of its query rows.
template <int D, int NG>
struct Query {
  uint32_t b[D / 32][4];  // B fragments of S^T: head gid, the channels of this lane's K words
  uint32_t zero;          // B fragment of the zeros' part: part tig of scale * sum q, by group
  float xs[2];            // the scores' factor, of heads 2 tig and 2 tig + 1
};

// Two runs of 16 keys, at rec0 and rec1 (records, or a record and its second half of rows): two, so that
// their dependent steps overlap. kTail: only the first `valid` of the 32 keys count, and whatever the other
// slots hold (NaN too) is taken out of the products.
template <int D, int NG, int BS, bool kTail>
ES_DEVICE void attend(Acc<D, NG>& A, const Query<D, NG>& Q, bool first, const uint8_t* rec0, const uint8_t* rec1,
                      int sub1, int gid, int tig, int valid) {
  using R = Rec<D, NG, BS>;
  constexpr int KW = D / 32, VW = D / 64, MT = D / 16;
  const int kr = key_of_row(gid);
  // S^T = K . q^T on the codes
  uint32_t kw[2][2][KW];  // [run][row gid | gid + 8][word]
  uint32_t kp[2][2][NG], vp[2][2][NG];
#pragma unroll
  for (int u = 0; u < 2; u++) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int row = (u ? sub1 : 0) * 16 + 8 * i + kr;
      const uint8_t* rec = u ? rec1 : rec0;
      const uint8_t* at = rec + row * R::kRow + tig * (D / 8);
      if (D == 128) {
        const uint4 w = *reinterpret_cast<const uint4*>(at);
        kw[u][i][0] = w.x, kw[u][i][1] = w.y, kw[u][i][KW - 2] = w.z, kw[u][i][KW - 1] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(at);
        kw[u][i][0] = w.x, kw[u][i][1] = w.y;
      }
      const uint8_t* mp = rec + R::kKMeta + row * R::kMeta;
      if (NG == 2) {
        const uint2 a = *reinterpret_cast<const uint2*>(mp);
        const uint2 b = *reinterpret_cast<const uint2*>(mp + BS * R::kMeta);
        kp[u][i][0] = a.x, kp[u][i][NG - 1] = a.y, vp[u][i][0] = b.x, vp[u][i][NG - 1] = b.y;
      } else {
        kp[u][i][0] = *reinterpret_cast<const uint32_t*>(mp);
        vp[u][i][0] = *reinterpret_cast<const uint32_t*>(mp + BS * R::kMeta);
      }
    }
  }
  float acc[2][NG][4];
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int g = 0; g < NG; g++) acc[u][g][0] = acc[u][g][1] = acc[u][g][2] = acc[u][g][3] = 0.f;
#pragma unroll
  for (int w = 0; w < KW; w++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float* d = acc[u][NG == 2 ? (w & 1) : 0];
      uint32_t wa = kw[u][0][w], wb = kw[u][1][w];
      const uint32_t a0[4] = {wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u};
      mma_f16_16816(d, a0, Q.b[w][0], Q.b[w][1]);
      wa >>= 8, wb >>= 8;
      const uint32_t a1[4] = {wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u, wb & 0x00F000F0u};
      mma_f16_16816(d, a1, Q.b[w][2], Q.b[w][3]);
    }
  // x[run][row i][head j] = score - m + k in the log2 domain
  float x[2][2][2];
  float top[2] = {-INFINITY, -INFINITY}, smax = 0.f;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    float z[4];
    // (one group: the scale in the low half meets a zero of B)
    if (NG == 2)
      mma_bf16_1688(z, __byte_perm(kp[u][0][0], kp[u][0][NG - 1], 0x7632), __byte_perm(kp[u][1][0], kp[u][1][NG - 1], 0x7632),
                    Q.zero, A.k - A.m[0], A.k - A.m[1]);
    else
      mma_bf16_1688(z, kp[u][0][0], kp[u][1][0], Q.zero, A.k - A.m[0], A.k - A.m[1]);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const bool in = !kTail || 16 * u + 8 * i + kr < valid;
      float t0 = pair_scale(kp[u][i][0]) * acc[u][0][2 * i], t1 = pair_scale(kp[u][i][0]) * acc[u][0][2 * i + 1];
      if (NG == 2) {
        t0 = fmaf(pair_scale(kp[u][i][NG - 1]), acc[u][NG - 1][2 * i], t0);
        t1 = fmaf(pair_scale(kp[u][i][NG - 1]), acc[u][NG - 1][2 * i + 1], t1);
      }
#pragma unroll
      for (int g = 0; g < NG; g++) {
        if (!in) vp[u][i][g] = 0;
        smax = fmaxf(smax, pair_scale(vp[u][i][g]));
      }
      x[u][i][0] = in ? fmaf(t0, Q.xs[0], z[2 * i]) : -INFINITY;
      x[u][i][1] = in ? fmaf(t1, Q.xs[1], z[2 * i + 1]) : -INFINITY;
      top[0] = fmaxf(top[0], x[u][i][0]);
      top[1] = fmaxf(top[1], x[u][i][1]);
    }
  }
  if (__any_sync(0xffffffffu, first || fmaxf(top[0], top[1]) > A.k + kSlack || smax > A.vlim)) {
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], s));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], s));
      smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, s));
    }
    float dk = 0.f;  // what k falls by
    if (smax > A.vlim) {
      const int e = exponent(smax) + 1;
      const float k = (float)(kPBits - e);
      dk = A.k - k;
      A.k = k;
      A.vlim = pow2i(e + 2);
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
      // the maximum: of the first keys as it is (none of them counted: left where it is), later the larger
      const float up = top[j] - (A.k + dk);
      const float dm = first ? (up == -INFINITY ? 0.f : up) : fmaxf(up, 0.f);
      A.m[j] += dm;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 2; i++) x[u][i][j] -= dm + dk;
      const float c = ex2(-(dm + dk));
      if (!first) {
        A.l[j] *= c;
#pragma unroll
        for (int g = 0; g < NG; g++) A.zs[j][g] *= c;
#pragma unroll
        for (int i = 0; i < MT; i++) A.o[i][j] *= c, A.o[i][2 + j] *= c;
      }
    }
  }
  // P, its sums, and P * scale as the B fragments of O^T (keys along k): transposed in registers
  uint32_t pb[2][NG][2];
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float p0 = ex2(x[u][i][0]), p1 = ex2(x[u][i][1]);
      A.l[0] += p0;
      A.l[1] += p1;
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const float z = pair_zero(vp[u][i][g]), s = pair_scale(vp[u][i][g]);
        A.zs[0][g] = fmaf(p0, z, A.zs[0][g]);
        A.zs[1][g] = fmaf(p1, z, A.zs[1][g]);
        pb[u][g][i] = transpose8(pack_f16x2(p0 * s, p1 * s));
      }
    }
  // O^T += V^T . P^T on the codes: rows gid and gid + 8 of tile (w, j) are channels 2 j and 2 j + 1 of
  // word w, a register's halves the keys of rows 2 tig and 2 tig + 1. (Leaving the even j a whole byte, c_j +
  // 16 c_{j + 1}, and subtracting in the end saves a mask in six, but the tensor core's sums truncate, and
  // what 128K keys average to is 1/100 of their codes' sum: seventeen times the bias showed as 0.6%.)
#pragma unroll
  for (int u = 0; u < 2; u++) {
    uint32_t v[4][VW];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int row = (u ? sub1 : 0) * 16 + 8 * (j >> 1) + ((j & 1) ? (tig ^ 1) + 4 : tig);
      const uint8_t* at = (u ? rec1 : rec0) + R::kV + row * R::kRow + gid * (D / 16);
      if (D == 128) {
        const uint2 w = *reinterpret_cast<const uint2*>(at);
        v[j][0] = w.x, v[j][VW - 1] = w.y;
      } else {
        v[j][0] = *reinterpret_cast<const uint32_t*>(at);
      }
    }
#pragma unroll
    for (int w = 0; w < VW; w++) {
      const int g = NG == 2 ? w : 0;
      uint32_t r[4] = {__byte_perm(v[0][w], v[1][w], 0x5410), __byte_perm(v[0][w], v[1][w], 0x7632),
                       __byte_perm(v[2][w], v[3][w], 0x5410), __byte_perm(v[2][w], v[3][w], 0x7632)};
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t a0[4], a1[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          a0[e] = r[e] & 0x000F000Fu;
          a1[e] = r[e] & 0x00F000F0u;
          r[e] >>= 8;
        }
        mma_f16_16816(A.o[w * 4 + 2 * h], a0, pb[u][g][0], pb[u][g][1]);
        mma_f16_16816(A.o[w * 4 + 2 * h + 1], a1, pb[u][g][0], pb[u][g][1]);
      }
    }
  }
}

// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a row's splits. A row of at most kFew splits is one
// warp's, in order; a longer one is a CTA's: warp w takes splits w, w + 8, ..., then the warps add in order.
// (The rule is the row's own count, so its bits do not depend on the launch.) Four splits' loads are on the
// way at a time.
constexpr int kMergeWarps = 8;
constexpr int kFew = 16;

template <int D>
struct Part {
  static constexpr int E = D / 32;  // neighbouring channels of a lane
  float acc[E], l;
  // splits first, first + step, ... of a row whose maximum is mx; po(i), ml(i): split i's output and (m, l)
  template <typename O, typename M>
  ES_DEVICE void sum(O&& po, M&& ml, int ns, int first, int step, float mx, int lane) {
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = 0.f;
#pragma unroll 4
    for (int i = first; i < ns; i += step) {
      const float2 t = ml(i);
      const float f = t.x == mx ? 1.f : ex2(t.x - mx);
      l = fmaf(t.y, f, l);
      float v[E];
      if (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(po(i) + E * lane);
        v[0] = x.x, v[1] = x.y, v[E - 2] = x.z, v[E - 1] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(po(i) + E * lane);
        v[0] = x.x, v[1] = x.y;
      }
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] = fmaf(v[e], f, acc[e]);
    }
  }
  ES_DEVICE void write(__nv_bfloat16* out, int lane) const {
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<__nv_bfloat162*>(out + E * lane + e) = __floats2bfloat162_rn(acc[e] / l, acc[e + 1] / l);
  }
};

template <int D, int NG, int BS>
__global__ void __launch_bounds__(kDecThreads, kDecCtas) decode_kernel(DecodeParams p) {
  using R = Rec<D, NG, BS>;
  using C = Ring<D, NG, BS>;
  constexpr int KW = D / 32;  // K words a lane holds of a key
  constexpr int VW = D / 64;  // V words
  constexpr int PB = C::kStep, ST = C::kSteps;
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
  float* own_o = reinterpret_cast<float*>(ring);  // [8][D] and (m, l) [8], once the ring is done with
  if (lane == 0) {
    for (int i = 0; i < ST; i++) ptx::mbar_init(&full[i], 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();

  pdl_wait();
  pdl_launch();
  const int ctx = min(p.ctx_lens[b], p.bt_cols * BS);
  const int ns = min(p.max_splits, splits_of(ctx));
  const int64_t row0 = (int64_t)b * p.hq + head0;
  auto attend_split = [&]() {
    if (ctx <= 0) {
      if (split == 0)  // an empty history: the output is zero
        for (int i = lane; i < heads * D; i += 32) p.out[((int64_t)b * p.hq + head0) * D + i] = f2bf(0.f);
      return;
    }
    const int plen = ((ctx + ns - 1) / ns + BS - 1) / BS * BS;  // equal splits, to a block
    const int s0 = split * plen, s1 = min(ctx, s0 + plen);
    if (split >= ns) return;
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
    int issued = 0;  // blocks whose copies are on the way or done
    auto issue = [&](int stage) {  // the next step's
      if (issued != 0 && (issued & 31) == 0) ids = entries(issued);
      const int n = min(PB, blocks - issued);
      const int64_t b0 = __shfl_sync(0xffffffffu, ids, issued & 31), b1 = __shfl_sync(0xffffffffu, ids, (issued + PB - 1) & 31);
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(&full[stage], n * R::kBytes);
        uint8_t* dst = ring + stage * PB * R::kBytes;
        ptx::bulk_g2s_hint(dst, head_base + b0 * p.s_block, R::kBytes, &full[stage], pol);
        if (n == 2) ptx::bulk_g2s_hint(dst + R::kBytes, head_base + b1 * p.s_block, R::kBytes, &full[stage], pol);
      }
      issued += n;
    };
    for (int i = 0; i < ST && issued < blocks; i++) issue(i);

    // the query, scaled to <= 2^10
    Query<D, NG> Q;
    {
      float qv[KW][8];
      float qmax = 0.f, sum[2] = {0.f, 0.f};
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
          sum[NG == 2 ? (w & 1) : 1] += qv[w][i];
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, o));
#pragma unroll
        for (int g = 0; g < 2; g++) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], o);
      }
      const int e = exponent(qmax);
      const float f = pow2i(9 - e), f16th = f * 0.0625f;
#pragma unroll
      for (int w = 0; w < KW; w++) {
        Q.b[w][0] = pack_f16x2(qv[w][0] * f, qv[w][1] * f);
        Q.b[w][1] = pack_f16x2(qv[w][2] * f16th, qv[w][3] * f16th);
        Q.b[w][2] = pack_f16x2(qv[w][4] * f, qv[w][5] * f);
        Q.b[w][3] = pack_f16x2(qv[w][6] * f16th, qv[w][7] * f16th);
      }
      const float x = p.scale_log2 * pow2i(24 - 9 + e);
#pragma unroll
      for (int i = 0; i < 2; i++) Q.xs[i] = __shfl_sync(0xffffffffu, x, (2 * tig + i) * 4);
      // scale * sum q in three terms of 8 bits, lane tig the tig-th: (first group, second), or with one group
      // (0, the sum), which meets (scale, zero) of a key as stored
      float t[2] = {p.scale_log2 * sum[0], p.scale_log2 * sum[1]};
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (i < tig) t[0] -= bf2f(f2bf(t[0])), t[1] -= bf2f(f2bf(t[1]));
      Q.zero = tig < 3 ? ptx::pack_bf16x2(t[0], t[1]) : 0u;
    }

    Acc<D, NG> A;
#pragma unroll
    for (int i = 0; i < D / 16; i++) A.o[i][0] = A.o[i][1] = A.o[i][2] = A.o[i][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      A.m[j] = 0.f, A.l[j] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; g++) A.zs[j][g] = 0.f;
    }
    A.k = 0.f;
    A.vlim = 0.f;

    int stage = 0, phase = 0;
    for (int i = 0; i < blocks; i += PB) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[stage], phase))) {
        // the copies on their way have to land before the warp leaves
        for (int k = i / PB; k * PB < issued; k++) ptx::mbar_wait(&full[k % ST], (k / ST) & 1);
        if (lane == 0 && p.status) atomicExch(p.status, (int)kTimeout);
        return;
      }
      const uint8_t* rec0 = ring + stage * PB * R::kBytes;
      const uint8_t* rec1 = PB == 2 ? rec0 + R::kBytes : rec0;  // (of a block the split lacks: not counted)
      const int valid = s1 - s0 - i * BS;
      if (valid >= 32)
        attend<D, NG, BS, false>(A, Q, i == 0, rec0, rec1, 2 - PB, gid, tig, 32);
      else
        attend<D, NG, BS, true>(A, Q, i == 0, rec0, rec1, 2 - PB, gid, tig, valid);
      __syncwarp();  // every lane has read the step's stage
      if (issued < blocks) issue(stage);
      if (++stage == ST) stage = 0, phase ^= 1;
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
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int h = 2 * tig + j;
      if (h >= heads) continue;
      const float inv = 1.f / A.l[j];
#pragma unroll
      for (int w = 0; w < VW; w++) {
        float y[8];  // channels 8 (gid + 8 w) and up
        const float z = A.zs[j][NG == 2 ? w : 0];
#pragma unroll
        for (int i = 0; i < 4; i += 2)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float even = A.o[w * 4 + i][2 * c + j], odd = A.o[w * 4 + i + 1][2 * c + j];
            y[2 * i + c] = fmaf(even, 16777216.f, z);         // 2^24: a code in bits 0..3
            y[2 * i + 2 + c] = fmaf(odd, 1048576.f, z);       // 2^20: in bits 4..7
          }
        const int ch = 8 * (gid + 8 * w);
        if (ns == 1) {
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] *= inv;
          *reinterpret_cast<uint4*>(p.out + (row0 + h) * D + ch) = pack8(y);
        } else {
          float4* po = reinterpret_cast<float4*>(p.join ? own_o + h * D + ch : p.part_o + ((row0 + h) * p.max_splits + split) * D + ch);
          po[0] = make_float4(y[0], y[1], y[2], y[3]);
          po[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
      if (ns > 1 && gid == 0)
        *(p.join ? reinterpret_cast<float2*>(own_o + 8 * D) + h
                 : reinterpret_cast<float2*>(p.part_ml) + (row0 + h) * p.max_splits + split) = make_float2(A.m[j] - A.k, A.l[j]);
    }
  };
  attend_split();
  if (!p.join || ctx <= 0 || ns == 1) return;
  // the splits' results, in the warps' own rings, joined a warp a query head
  __syncthreads();
  for (int h = warp; h < heads; h += kDecWarps) {
    Part<D> a;
    auto ml = [&](int i) { return reinterpret_cast<const float2*>(smem + i * C::kBytes + 8 * D * 4)[h]; };
    const float mx = warp_max(lane < ns ? ml(lane).x : -INFINITY);
    a.sum([&](int i) { return reinterpret_cast<const float*>(smem + i * C::kBytes) + h * D; }, ml, ns, 0, 1, mx, lane);
    a.write(p.out + (row0 + h) * D, lane);
  }
}

// kRows: a CTA takes kMergeWarps rows, a warp each (no row has more than kFew splits); else one row.
template <int D, bool kRows>
__global__ void __launch_bounds__(kMergeWarps * 32)
    merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ ctx_lens,
                 __nv_bfloat16* __restrict__ out, int64_t rows, int hq, int max_splits, int max_keys) {
  constexpr int E = D / 32;
  __shared__ float so[kRows ? 1 : kMergeWarps][D], sl[kMergeWarps], smx[kMergeWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = kRows ? (int64_t)blockIdx.x * kMergeWarps + warp : blockIdx.x;
  pdl_wait();
  pdl_launch();
  if (row >= rows) return;
  const int ns = min(max_splits, splits_of(min(ctx_lens[row / hq], max_keys)));
  if (ns <= 1) return;  // written by the split itself
  auto ml = [&](int i) { return reinterpret_cast<const float2*>(part_ml)[row * max_splits + i]; };
  auto po = [&](int i) { return part_o + (row * max_splits + i) * D; };
  Part<D> a;
  if (ns <= kFew) {
    if (!kRows && warp > 0) return;
    const float mx = warp_max(lane < ns ? ml(lane).x : -INFINITY);
    a.sum(po, ml, ns, 0, 1, mx, lane);
    a.write(out + row * D, lane);
    return;
  }
  if (kRows) return;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < ns; i += kMergeWarps * 32) mx = fmaxf(mx, ml(i).x);
  mx = warp_max(mx);
  if (lane == 0) smx[warp] = mx;
  __syncthreads();
  mx = smx[0];
#pragma unroll
  for (int w = 1; w < kMergeWarps; w++) mx = fmaxf(mx, smx[w]);
  a.sum(po, ml, ns, warp, kMergeWarps, mx, lane);
#pragma unroll
  for (int e = 0; e < E; e++) so[warp][E * lane + e] = a.acc[e];
  if (lane == 0) sl[warp] = a.l;
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
  if (e != cudaSuccess || p.join) return e;
  const int64_t rows = (int64_t)B * p.hq;
  auto merge = [&](auto kernel, int64_t grid) {
    return launch_ex(kernel, dim3((unsigned)grid), dim3(kMergeWarps * 32), 0, stream, 0, (const float*)p.part_o,
                     (const float*)p.part_ml, p.ctx_lens, p.out, rows, p.hq, p.max_splits, p.bt_cols * BS);
  };
  return p.max_splits <= kFew ? merge(merge_kernel<D, true>, (rows + kMergeWarps - 1) / kMergeWarps)
                              : merge(merge_kernel<D, false>, rows);
}

}  // namespace kv4

bool kv4_decode_joins(int64_t max_splits) { return max_splits <= kv4::kDecWarps; }

int64_t kv4_max_splits(int64_t max_len) {
  // the most of any length up to max_len: the count falls where the splits get longer
  const int n = (int)std::min<int64_t>(max_len, INT32_MAX - 1024);
  int most = kv4::splits_of(n);
  if (n > 1024) most = std::max(most, kv4::splits_of(1024));
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
  p.join = a.max_splits <= kv4::kDecWarps;
  p.scale_log2 = a.scale * kv4::kLog2eF;
  if ((int64_t)p.hkv * p.head_tiles > 65535 || (int64_t)a.B * a.hq > INT32_MAX) return cudaErrorInvalidValue;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    return kv4::launch_decode<d, ng, bs>(p, a.B, stream);
  });
}

}  // namespace es
