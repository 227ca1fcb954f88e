// Causal attention of a step's new rows over their sequences' paged history held in 4 bits (tcgen05, TMEM).
//
// The products are large here (128 and more query rows share a key), so a key's codes are turned into
// f16 values once for 256 query rows and the tensor cores do the rest: v = scale * c + zero, c exact in
// f16 and the multiply-add rounded once. The query rows of one kv head's whole group are packed into the
// rows of a tile (row = token * G + head of the group), so grouped heads share the conversion too.
//
// f16 carries 11 bits where bf16 carries 8 (a key in bf16 alone would double the error of the output), but
// fewer exponents. So each operand stands under a power of two of its own: a query row's, which its scores'
// factor takes back; a key tile's of K, likewise; and a key tile's of V, which enters the exponent of that
// tile's probabilities against the largest so far. None of them costs an operation per element.
//
// A CTA keeps to its SM and walks work items: 256 rows (two tiles of 128) of one sequence and kv head,
// over a run of 128-key tiles. Its warps:
//   * 8-11 turn tile j's codes (loaded a tile ahead, straight to registers) into K and V stages in shared
//     memory, 128-byte swizzled, each freed by itself: K's by the second S, so that the next keys are there
//     while this tile's softmax runs (one barrier for both: 711 us for the 8192-row prompt);
//   * 12 issues the MMAs: S_t = Q_t . K_j^T and O_t += P_t . V_j for t = 0, 1 in turn, P read from TMEM;
//   * 0-3 and 4-7 do the softmax of tiles 0 and 1, a thread a row: S from TMEM, P back over it in f16, the
//     first half of it for the tensor core to start on (P as a whole: 16 prompts 136 us instead of 131).
// While one tile's softmax runs, the tensor core works for the other. The running maximum moves (and O in
// TMEM is rescaled) only when a score passes it by 2^6, so most tiles leave O alone. A row's sums are fp32.
// Registers go where they are needed: 184 a softmax thread (a row's 128 scores at once), 104 a converting one.
//
// A sequence with few rows and a long history is cut along its keys as well, into items whose results
// (O, m, l) a second kernel joins. The cut depends on the sequence's own rows and keys and on the model's
// heads, never on the batch. An item is found by a scan over the sequences, so the host needs no plan and no
// synchronisation; a warp of each CTA hands items out ahead of their readers. All waits are bounded and end in
// the status word.
//
// Measured (32 / 8 heads of 128): one prompt of 8192 rows in 605-632 us, 870-910 TFLOP/s, half of what cuBLAS
// reaches.
// A key tile takes 4,300 cycles where its 32 MMAs need 2,060 and its exponentials 2,050: each query tile's chain
// S -> softmax -> P -> MMAs is longer than the two tiles' overlap hides, and the conversion's stores and the MMAs
// share the shared memory's bandwidth. (An eighth of the exponentials as polynomials on the FMA pipe: slower,
// 654 us; instructions bound the softmax, not the exponential unit.) 16 prompts of 8191 rows in all take 121 us:
// an item of three key tiles pays as much again for its query, its first conversion and its output. Two more
// warps that copied the next item's query ahead made that 130 us.
#include <algorithm>
#include <atomic>
#include <climits>

#include "api.h"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace es {
namespace kv4 {

constexpr int kRows = 128;  // rows of a tile (MMA M)
constexpr int kKeys = 128;  // keys of a tile (MMA N of S, K of P.V)
constexpr int kSoftThreads = 256;
constexpr int kConvThreads = 128;
constexpr int kPreThreads = kSoftThreads + kConvThreads + 128;  // (the MMA warp's group: kMmaRegs)
constexpr int kSoftRegs = 184, kConvRegs = 104, kMmaRegs = 40;
static_assert(kSoftRegs * kSoftThreads + kConvRegs * kConvThreads + kMmaRegs * 128 <= 128 * kPreThreads,
              "the split draws on the registers of the launch, 128 a thread");
constexpr int kTmem = 512;  // S0, S1 (128 columns each, P over them), O0, O1

// Wait for phase `parity` of `bar`: at most 2^20 tries of up to 2 us each. (Reading the global timer for the bound
// is more code at each of 16 places, which warps in different roles fetch at once: 122.4 us for 16 prompts.)
ES_DEVICE bool wait_for(uint64_t* bar, uint32_t parity) {
  for (uint32_t tries = 0; tries < (1u << 20); tries++)
    if (ptx::mbar_try_wait(bar, parity, 2000u)) return true;
  return false;
}

template <int D>
struct PreCfg {
  static constexpr int kChunk = kRows * 128;           // one 64-channel chunk of a 128-row operand
  static constexpr int kTile = (D / 64) * kChunk;      // an f16 tile of 128 rows
  static constexpr int kSmem = 1024 + 2 * kTile + 2 * 2 * kTile + 256;
};

constexpr float kPreSlack = 6.f;  // log2 of how far a score may pass the running maximum
constexpr float kPreBits = 9.f;   // P enters f16 as at most 2^(6 + 9)
constexpr int kFirst = 2;         // quarters of a tile's P that the tensor core takes while the rest is computed
constexpr int kTop = 13;          // operands are scaled to below 2^(kTop + 1)

template <int N>
ES_DEVICE void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
ES_DEVICE void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct PreParams {
  const __nv_bfloat16* q;  // [T, hq, D] rows of q_stride
  int64_t q_stride;
  const uint8_t* cache;
  int64_t s_block, num_blocks;
  const int* block_tables;
  int64_t bt_stride;
  int bt_cols;
  const int* ctx_lens;
  const int64_t* last_rows;
  __nv_bfloat16* out;  // [T, hq, D]
  float* part_o;       // [parts * hq, D]: a row's parts head by head
  float* part_ml;      // [parts * hq, 2]
  uint2* part_at;      // [T]: (its parts | its sequence's << 16, its first part's row); null: nothing is cut
  int* status;
  unsigned* next;      // items handed out beyond each CTA's first, zero before the launch
  int T, S, hq, hkv, G, tt;  // tt: tokens of a 128-row tile
  int parts;                 // rows times splits that the workspace holds
  float scale_log2;
};

// How a sequence of `tiles` row tiles and `keys` key tiles is cut along its keys: the key tiles of an item, and the
// items that a row tile has at most. Not at all where its row tiles fill the SMs; else into kCutItems items at most, which
// bounds its parts in the workspace whatever its length (256 rows of a head an item: 34 to 51 MB at head dim 128).
// (64 rows on 131K keys, 32 / 8 heads of 128: 203 us, without the bound 245; 900 rows on 60K: 1,265 and 1,237; 509
// rows on 0-40K keys, 14 / 2 of 64: 106 and 107.)
struct Cut {
  int chunk, splits;
};
constexpr int kCutItems = 256;
__host__ __device__ __forceinline__ int least_chunk(int items) { return items > 16 ? 16 : 8; }
__host__ __device__ __forceinline__ int most_splits(int items) { return (kCutItems + items - 1) / items; }
__host__ __device__ __forceinline__ Cut cut_of(int tiles, int hkv, int keys) {
  const int items = tiles * hkv;
  Cut c{1 << 24, 1};
  if (items == 0 || items >= 128 || keys <= 0) return c;
  const int least = least_chunk(items), most = most_splits(items), fair = (keys + most - 1) / most;
  c.chunk = least > fair ? least : fair;
  c.splits = (keys + c.chunk - 1) / c.chunk;
  return c;
}

struct Item {
  int seq, rows, row0, ctx;  // the sequence, its rows, its first row, its context length
  int tile, head, split, chunk;
  int j0, j1, ns;  // its key tiles, and how many items its row tile has
  int per, part0;  // the sequence's splits, and its first row in the workspace
};

// Work item `idx`, in an order that puts long ones first: of 32 sequences at a time those with the most keys,
// of a sequence its last tiles. False: there is none. The whole warp calls it.
ES_DEVICE bool find_item(const PreParams& p, int bs, int idx, Item& it) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  int64_t parts = 0;  // of the sequences before these 32
#pragma unroll 1
  for (int s0 = 0; s0 < p.S; s0 += 32) {
    const int s = s0 + lane;
    int rows = 0, r0 = 0, ctx = 0, tiles = 0, ns = 0, chunk = 1, items = 0;
    if (s < p.S) {
      const int64_t T = p.T;
      r0 = s == 0 ? 0 : (int)max((int64_t)0, min(T, p.last_rows[s - 1] + 1));
      rows = max(0, (int)min(T, p.last_rows[s] + 1) - r0);
      ctx = min(p.ctx_lens[s], p.bt_cols * bs);
      tiles = (rows + 2 * p.tt - 1) / (2 * p.tt);
      const Cut c = cut_of(tiles, p.hkv, (ctx + kKeys - 1) / kKeys);
      chunk = c.chunk, ns = c.splits;
    }
    // its place in the workspace; one that the workspace has no room for is not cut
    int part0 = 0;
    if (p.parts > 0) {
      const int need = ns > 1 ? rows * ns : 0;
      int sum = need;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      part0 = (int)min(parts + sum - need, (int64_t)p.parts);
      if (parts + sum > p.parts) chunk = 1 << 24, ns = 1;
      parts += __shfl_sync(0xffffffffu, sum, 31);
    } else {
      chunk = 1 << 24, ns = 1;
    }
    items = tiles * ns * p.hkv;
    // this lane's place in the order: the sequence (lane) `src`
    int src = lane;
    if (p.S > 1) {
      int rank = 0;
#pragma unroll 1
      for (int k = 0; k < 32; k++) {
        const int c = __shfl_sync(0xffffffffu, ctx, k);
        rank += c > ctx || (c == ctx && k < lane);
      }
#pragma unroll 1
      for (int k = 0; k < 32; k++)
        if (__shfl_sync(0xffffffffu, rank, k) == lane) src = k;
      items = __shfl_sync(0xffffffffu, items, src);
    }
    int upto = items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    if (idx < before + total) {
      const int place = __ffs(__ballot_sync(0xffffffffu, idx < before + upto)) - 1;
      const int first = before + __shfl_sync(0xffffffffu, upto - items, place);
      src = __shfl_sync(0xffffffffu, src, place);
      it.seq = s0 + src;
      it.rows = __shfl_sync(0xffffffffu, rows, src);
      it.row0 = __shfl_sync(0xffffffffu, r0, src);
      it.ctx = __shfl_sync(0xffffffffu, ctx, src);
      it.chunk = __shfl_sync(0xffffffffu, chunk, src);
      const int t = __shfl_sync(0xffffffffu, tiles, src), per = __shfl_sync(0xffffffffu, ns, src);
      it.per = per;
      it.part0 = __shfl_sync(0xffffffffu, part0, src);
      const uint32_t at = idx - first, group = at / (uint32_t)p.hkv, splits = (uint32_t)per;
      it.tile = t - 1 - (int)(group / splits);
      it.split = (int)(group % splits);
      it.head = (int)(at - group * p.hkv);
      return true;
    }
    before += total;
  }
  return false;
}

// The key tiles of an item, and how many items its row tile has.
ES_DEVICE void span(const PreParams& p, Item& it) {
  const int last = min(it.rows, (it.tile + 1) * 2 * p.tt) - 1;  // the tile's last token
  const int pos = min(it.ctx - it.rows + last, it.ctx - 1);
  const int J = pos < 0 ? 0 : pos / kKeys + 1;
  it.ns = max(1, (J - 1) / it.chunk + 1);
  it.j0 = it.split * it.chunk;
  it.j1 = it.split == it.ns - 1 ? J : min(J, it.j0 + it.chunk);
  if (it.split >= it.ns) it.j1 = it.j0;
}

// 8 codes -> 8 f16 values: a masked nibble under the exponent of 1024 (bits 0..3) or 64 (bits 4..7) is
// 1024 + c or 64 + c
ES_DEVICE uint4 values8(uint32_t w, __half2 s, __half2 z) {
  uint32_t r[4];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t lo = (w & 0x000F000Fu) | 0x64006400u, hi = (w & 0x00F000F0u) | 0x54005400u;
    const __half2 a = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&lo), __float2half2_rn(1024.f)), s, z);
    const __half2 b = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&hi), __float2half2_rn(64.f)), s, z);
    r[2 * h] = *reinterpret_cast<const uint32_t*>(&a);
    r[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&b);
    w >>= 8;
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// 2^e as a float, e in [-126, 127], and the exponent of a positive number (of its bits), clamped so that these
// factors stay normal numbers, and the product of a query row's and a key tile's does however small they are
// (a masked score's -infinity times zero would be NaN; large ones meet infinity where their scores pass fp32)
ES_DEVICE float pre_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
ES_DEVICE int pre_exponent(uint32_t bits) { return min(100, max(-40, (int)(bits >> 23) - 127)); }

// Where a converting thread reads: row tid / P of each pass of kConvThreads / P rows, piece tid % P of the
// row. A pass is a multiple of a block, so a thread stays at one row of its blocks.
template <int D, int NG, int BS>
struct Source {
  using R = Rec<D, NG, BS>;
  static constexpr int P = D / 32;
  const int* bt;        // the sequence's table, from this thread's first block of tile 0
  const uint8_t* base;  // this thread's piece of its row, in block 0
  uint32_t step;        // 16-byte units between blocks
  int first, ctx, piece;
  int64_t num_blocks;
  bool bad = false;  // met an entry that is not a block of this cache

  ES_DEVICE Source(const PreParams& p, const Item& it, int tid)
      : bt(p.block_tables + (int64_t)it.seq * p.bt_stride),
        base(p.cache + (int64_t)it.head * R::kBytes + tid / P % BS * R::kRow),
        step((uint32_t)(p.s_block >> 4)),
        first(tid / P),
        ctx(it.ctx),
        piece(tid % P),
        num_blocks(p.num_blocks) {}
  ES_DEVICE int key(int j, int i) const { return j * kKeys + i * (kConvThreads / P) + first; }
  ES_DEVICE int block(int j, int i) const { return key(j, i) < ctx ? bt[key(j, i) / BS] : 0; }
  // The codes and pairs of the i-th piece of tile j, side 0: K, 1: V (zero past the history, whatever the
  // slot holds: its values are zero then).
  ES_DEVICE void load(int j, int i, int blk, int side, uint4& codes, uint32_t* meta) {
    codes = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < NG; g++) meta[g] = 0;
    if (key(j, i) < ctx) {
      if ((uint32_t)blk >= (uint64_t)num_blocks) bad = true, blk = 0;
      const uint8_t* row = base + ((uint64_t)(uint32_t)blk * step << 4);
      codes = *reinterpret_cast<const uint4*>(row + side * R::kV + 16 * piece);
      const int off = first % BS;
      const uint32_t* m = reinterpret_cast<const uint32_t*>(row + R::kKMeta + side * BS * R::kMeta + off * (R::kMeta - R::kRow));
#pragma unroll
      for (int g = 0; g < NG; g++) meta[g] = m[g];
    }
  }
};

// The bits of a bound on a group's magnitudes; kNotFinite or more for a group that reads as NaN.
constexpr uint32_t kNotFinite = 0x7F800000u;
ES_DEVICE uint32_t bound_of(uint32_t pair) {
  const float z = pair_zero(pair);
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(z)), "f"(fabsf(fmaf(15.f, pair_scale(pair), z))));
  return __float_as_uint(d);
}

// One piece of row `row` into a tile's swizzled layout, times f.
template <int D, int NG>
ES_DEVICE void store_piece(uint8_t* tile, int row, int piece, const uint4& codes, const uint32_t* meta, float f) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  __half2 s[NG], z[NG];
#pragma unroll
  for (int g = 0; g < NG; g++) {
    s[g] = __float2half2_rn(pair_scale(meta[g]) * f);
    z[g] = __float2half2_rn(pair_zero(meta[g]) * f);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int chunk = D == 128 ? (i & 1) : 0;
    const int unit = D == 128 ? 2 * piece + (i >> 1) : 4 * piece + i;
    const int g = NG == 2 ? chunk : 0;
    *reinterpret_cast<uint4*>(tile + chunk * PreCfg<D>::kChunk + row * 128 + ((unit ^ (row & 7)) << 4)) =
        values8(w[i], s[g], z[g]);
  }
}

template <int D, int NG, int BS>
__global__ void __launch_bounds__(kPreThreads, 1) prefill_kernel(PreParams p) {
  using C = PreCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                  // [2] tiles
  uint8_t* kv_s = smem + 2 * C::kTile;  // [2] stages of K tile, V tile
  uint64_t* bar = reinterpret_cast<uint64_t*>(kv_s + 4 * C::kTile);
  uint64_t *q_full = bar, *s_full = bar + 2, *p_full = bar + 4, *o_full = bar + 6;
  uint64_t *k_full = bar + 8, *k_empty = bar + 10, *v_full = bar + 12, *v_empty = bar + 14;
  uint64_t* mma_done = bar + 16;
  uint64_t *item_full = bar + 17, *item_empty = bar + 19;
  uint64_t* p_part = bar + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 23);
  __shared__ int s_fail;
  __shared__ Item s_item[2];             // items ahead of their readers; seq -1: there is none
  __shared__ uint32_t s_bound[2][2][4];  // [tile parity][K, V][converting warp]: largest magnitudes' bits
  __shared__ int s_exp[4][2];            // [tile & 3][K, V]: the tile's exponents
  __shared__ int s_nan[4][NG];           // [item & 3][group]: the item's first key whose V reads as NaN

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_fail = 0;
    for (int i = 0; i < 2; i++) {
      ptx::mbar_init(&item_full[i], 1);
      ptx::mbar_init(&item_empty[i], 13);  // a lane of every warp that reads items
      ptx::mbar_init(&q_full[i], 128);
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&p_part[i], 128);
      ptx::mbar_init(&p_full[i], 128);
      ptx::mbar_init(&o_full[i], 1);
      ptx::mbar_init(&k_full[i], kConvThreads);
      ptx::mbar_init(&k_empty[i], 1);
      ptx::mbar_init(&v_full[i], kConvThreads);
      ptx::mbar_init(&v_empty[i], 1);
    }
    ptx::mbar_init(mma_done, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 12) ptx::tmem_alloc(tmem_slot, kTmem);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch();

  Item it;
  bool ok = true;
  // The warp's next item, in order, into `it` (false: none, or a wait ran out).
  uint32_t taken = 0;
  auto next_item = [&]() {
    const int s = taken & 1;
    ok = __all_sync(0xffffffffu, wait_for(&item_full[s], (taken >> 1) & 1)) && ok;
    if (!ok) return false;
    it = s_item[s];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&item_empty[s]);
    taken++;
    return it.seq >= 0;
  };
  if (warp >= 8 && warp < 12) {
    // ---- codes to values ------------------------------------------------------------------------
    regs_down<kConvRegs>();
    constexpr int P = D / 32;
    const int tid = threadIdx.x - kSoftThreads;
    uint32_t n = 0, items = 0;  // key tiles converted so far, over all items; items with any
    bool left = false;
    if (tid < NG) s_nan[0][tid] = INT_MAX;
    while (!left) {
      const bool any = next_item();
      left = ptx::named_bar_or(1, kConvThreads, !ok);  // where a wait of one of the converting warps ran out, all leave
      if (left || !any) break;
      if (it.j0 >= it.j1) continue;
      Source<D, NG, BS> src(p, it, tid);
      uint4 kc[P], vc[P];  // the next tile's codes and pairs
      uint32_t km[P][NG], vm[P][NG];
      int blk[P];  // and its blocks: a table entry is asked for two tiles ahead, its data one
      int vr = -100;  // the largest of V's exponents so far
#pragma unroll
      for (int i = 0; i < P; i++) blk[i] = src.block(it.j0, i);
#pragma unroll
      for (int i = 0; i < P; i++) {
        src.load(it.j0, i, blk[i], 0, kc[i], km[i]);
        src.load(it.j0, i, blk[i], 1, vc[i], vm[i]);
        blk[i] = src.block(it.j0 + 1, i);
      }
#pragma unroll 1
      for (int j = it.j0; j < it.j1; j++, n++) {
        const int s = n & 1;
        uint8_t* kt = kv_s + s * 2 * C::kTile;
        // the tile's largest magnitudes over the converting warps, whose barrier is where they leave together
        uint32_t kb = 0, vb = 0;
#pragma unroll
        for (int i = 0; i < P; i++)
#pragma unroll
          for (int g = 0; g < NG; g++) kb = max(kb, bound_of(km[i][g])), vb = max(vb, bound_of(vm[i][g]));
        kb = __reduce_max_sync(0xffffffffu, kb);
        vb = __reduce_max_sync(0xffffffffu, vb);
        if (__builtin_expect(max(kb, vb) >= kNotFinite, 0)) {
          // A group that reads as NaN sets no exponent. K's stays in its key's scores, which a mask replaces; V's
          // would reach every row of the tile through a probability of zero, so it counts as zero here, and the
          // rows that see its key, or a later one, get their NaN in the end.
          kb = vb = 0;
#pragma unroll
          for (int i = 0; i < P; i++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
              const uint32_t k = bound_of(km[i][g]), v = bound_of(vm[i][g]);
              if (k < kNotFinite) kb = max(kb, k);
              if (v < kNotFinite) {
                vb = max(vb, v);
              } else {
                vm[i][g] = 0;
                atomicMin(&s_nan[items & 3][g], src.key(j, i));
              }
            }
          kb = __reduce_max_sync(0xffffffffu, kb);
          vb = __reduce_max_sync(0xffffffffu, vb);
        }
        if (lane == 0) s_bound[s][0][warp - 8] = kb, s_bound[s][1][warp - 8] = vb;
        if (n >= 2) ok = __all_sync(0xffffffffu, wait_for(&k_empty[s], ((n >> 1) - 1) & 1)) && ok;
        left = ptx::named_bar_or(1, kConvThreads, !ok);
        if (left) break;
        const uint32_t *bk = s_bound[s][0], *bv = s_bound[s][1];
        kb = max(max(bk[0], bk[1]), max(bk[2], bk[3]));
        vb = max(max(bv[0], bv[1]), max(bv[2], bv[3]));
        const int ke = pre_exponent(kb);
        // (not far below the largest: a tile of small values leaves its probabilities' range alone)
        const int ve = max(pre_exponent(vb), vr - 20);
        vr = max(vr, ve);
        if (tid == 0) s_exp[n & 3][0] = ke, s_exp[n & 3][1] = ve;
        const float kf = pre_pow2(kTop - ke), vf = pre_pow2(kTop - ve);
        const bool on = j + 1 < it.j1;
#pragma unroll
        for (int i = 0; i < P; i++) {
          store_piece<D, NG>(kt, i * (kConvThreads / P) + tid / P, tid % P, kc[i], km[i], kf);
          if (on) src.load(j + 1, i, blk[i], 0, kc[i], km[i]);
        }
        ptx::fence_proxy_async();
        ptx::mbar_arrive(&k_full[s]);
        if (n >= 2) ok = __all_sync(0xffffffffu, wait_for(&v_empty[s], ((n >> 1) - 1) & 1));
#pragma unroll
        for (int i = 0; i < P; i++) {
          store_piece<D, NG>(kt + C::kTile, i * (kConvThreads / P) + tid / P, tid % P, vc[i], vm[i], vf);
          if (on) {
            src.load(j + 1, i, blk[i], 1, vc[i], vm[i]);
            blk[i] = src.block(j + 2, i);
          }
        }
        ptx::fence_proxy_async();
        ptx::mbar_arrive(&v_full[s]);
      }
      // (the next entry, before the barrier ahead of its item: its last readers were the rows of the item three
      // before this one, and the query of the item after that has been asked for since)
      items++;
      if (tid < NG) s_nan[items & 3][tid] = INT_MAX;
      if (src.bad && p.status) atomicExch(p.status, (int)kBadShape);
    }
    if (!ok) s_fail = 1;
  } else if (warp >= 12) {
    // ---- MMA issuer, the warp that hands out items, and two that zero the rows of no sequence ---------
    regs_down<kMmaRegs>();
    if (warp == 13) {
      // An item's cost goes with its keys, so CTAs take their next one when they are ready for it, from one
      // counter (in turn: up to half of them waited for the longest, 16 prompts took 172 us).
      int idx = blockIdx.x;
      for (uint32_t k = 0; ok; k++) {
        const bool any = find_item(p, BS, idx, it);
        if (any) span(p, it);
        if (k >= 2) ok = __all_sync(0xffffffffu, wait_for(&item_empty[k & 1], ((k >> 1) - 1) & 1));
        if (!ok) break;
        if (lane == 0) {
          if (!any) it.seq = -1;
          s_item[k & 1] = it;
          ptx::mbar_arrive(&item_full[k & 1]);
        }
        if (!any) break;
        if (lane == 0) idx = (int)(gridDim.x + atomicAdd(p.next, 1u));
        idx = __shfl_sync(0xffffffffu, idx, 0);
      }
    }
    if (warp >= 14) {
      const int vecs = p.hq * (D / 8);
      for (int64_t x = max((int64_t)0, p.last_rows[p.S - 1] + 1) + blockIdx.x; x < p.T; x += gridDim.x) {
        uint4* row = reinterpret_cast<uint4*>(p.out) + x * vecs;
        for (int i = threadIdx.x & 63; i < vecs; i += 64) row[i] = make_uint4(0, 0, 0, 0);
        if ((threadIdx.x & 63) == 0 && p.part_at != nullptr) p.part_at[x] = make_uint2(1, 0);
      }
    }
    const bool failed = !ok;
    ok = warp == 12;
    constexpr uint32_t idesc_s = ptx::idesc_f16_f32(kRows, kKeys);
    constexpr uint32_t idesc_o = ptx::idesc_f16_f32(kRows, D) | (1u << 16);  // V: MN-major
    // The whole warp walks the loop, so that descriptors stay in uniform registers (a loop of one lane alone
    // spent 150 cycles an MMA on moving them there: 770 us for the 8192-row prompt); one lane issues, from
    // loops that stay rolled (unrolled they spilled, and their instructions had to be fetched anew each time).
    const bool leader = ptx::elect_one();
    const uint64_t q_desc = ptx::sw128_kmajor_desc(ptx::smem_u32(q_s)), k_desc = ptx::sw128_kmajor_desc(ptx::smem_u32(kv_s));
    const uint64_t v_desc = ptx::sw128_mnmajor_desc(ptx::smem_u32(kv_s + C::kTile), C::kChunk);
    constexpr int kStageStep = 2 * C::kTile >> 4;
    uint32_t n = 0, items = 0;
    auto qk = [&](int t, int s) {  // S_t = Q_t . K^T
      if (leader) {
        const uint64_t a = q_desc + t * (C::kTile >> 4), b = k_desc + s * kStageStep;
#pragma unroll 1
        for (int kk = 0; kk < D / 16; kk++) {
          const int off = (kk >> 2) * (C::kChunk >> 4) + 2 * (kk & 3);
          ptx::mma_f16_ss(tmem + t * 128, a + off, b + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        ptx::mma_commit(&s_full[t]);
        if (t == 1) ptx::mma_commit(&k_empty[s]);
      }
      __syncwarp();
    };
    while (ok && next_item()) {
      const int j0 = it.j0, j1 = it.j1;
      if (j0 >= j1) continue;
      ok = __all_sync(0xffffffffu, wait_for(&k_full[n & 1], (n >> 1) & 1));
      for (int t = 0; ok && t < 2; t++) {
        ok = __all_sync(0xffffffffu, wait_for(&q_full[t], items & 1));
        if (!ok) break;
        ptx::tc_fence_after();
        qk(t, n & 1);
      }
      for (int j = j0; ok && j < j1; j++, n++) {
        const int s = n & 1;
#pragma unroll 1
        for (int t = 0; t < 2; t++) {
          if (t == 0) ok = __all_sync(0xffffffffu, wait_for(&v_full[s], (n >> 1) & 1));
          const uint64_t b = v_desc + s * kStageStep;
          ok = ok && __all_sync(0xffffffffu, wait_for(&p_part[t], n & 1));
          if (!ok) break;
          ptx::tc_fence_after();
          if (leader) {
#pragma unroll 1
            for (int kk = 0; kk < 2 * kFirst; kk++)
              ptx::mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, b + kk * (16 * 128 >> 4), idesc_o,
                              (j > j0 || kk > 0) ? 1u : 0u);
          }
          __syncwarp();
          ok = __all_sync(0xffffffffu, wait_for(&p_full[t], n & 1));
          if (!ok) break;
          ptx::tc_fence_after();
          if (leader) {
#pragma unroll 1
            for (int kk = 2 * kFirst; kk < kKeys / 16; kk++)
              ptx::mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, b + kk * (16 * 128 >> 4), idesc_o,
                              (j > j0 || kk > 0) ? 1u : 0u);
            if (t == 1) ptx::mma_commit(&v_empty[s]);
            if (j + 1 == j1) ptx::mma_commit(&o_full[t]);
          }
          __syncwarp();
          if (j + 1 < j1) {
            if (t == 0) ok = __all_sync(0xffffffffu, wait_for(&k_full[s ^ 1], ((n + 1) >> 1) & 1));
            if (!ok) break;
            ptx::tc_fence_after();
            qk(t, s ^ 1);  // after P_t . V in the tensor core's order, which P_t's columns wait for
          }
        }
      }
      items++;
    }
    if (failed || (warp == 12 && !ok)) s_fail = 1;
    if (warp == 12) {
      if (leader) ptx::mma_commit(mma_done);
      __syncwarp();
      wait_for(mma_done, 0);  // nothing of this CTA is in flight past here
    }
  } else {
    // ---- softmax --------------------------------------------------------------------------------
    regs_up<kSoftRegs>();
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;  // row of the tile (TMEM lane)
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + t * 128 + lane_base, o_t = tmem + 256 + t * 128 + lane_base;
    const int inv_g = (65536 + p.G - 1) / p.G;  // x / G = (x * inv_g) >> 16 for x < 128
    const int token = (r * inv_g) >> 16, head = r - token * p.G;
    // This warp's 32 rows of the query tile, which no other warp touches: D / 8 lanes a row and 32 / U rows a
    // pass where memory is read or written, a thread a row where a row is scaled. unit(): 16-byte unit k of
    // row x in the tile's swizzled layout.
    constexpr int U = D / 8, kPass = 32 / U;
    const int w0 = (warp & 3) * 32;
    uint8_t* rows_s = q_s + t * C::kTile;
    auto unit = [&](int x, int k) {
      return reinterpret_cast<uint4*>(rows_s + (k >> 3) * C::kChunk + x * 128 + (((k & 7) ^ (x & 7)) << 4));
    };
    uint32_t n = 0, items = 0;
    while (ok && next_item()) {
      const int j0 = it.j0, j1 = it.j1, ns = it.ns;
      const int at = it.tile * 2 * p.tt + t * p.tt + token;
      const bool real = token < p.tt && at < it.rows;
      // where this thread's row is in memory: its elements of the query (-1: no row), its row of the output. The
      // lanes that move another's row ask it: a row of G heads takes a division and 64-bit products to find.
      const int64_t q_at = real ? (int64_t)(it.row0 + at) * p.q_stride + (it.head * p.G + head) * D : -1;
      const int64_t out_row = real ? (int64_t)(it.row0 + at) * p.hq + it.head * p.G + head : -1;
      const int pos = it.ctx - it.rows + at;
      // its place in the workspace: the row's parts, head by head
      const int part = ns > 1 ? (it.part0 + at * it.per) * p.hq + (it.head * p.G + head) * it.per + it.split : 0;
      if (real && it.split == 0 && it.head == 0 && head == 0 && p.part_at != nullptr)
        p.part_at[it.row0 + at] = ns > 1 ? make_uint2(ns | it.per << 16, it.part0 + at * it.per) : make_uint2(1, 0);
      if (j0 >= j1) {
        if (it.split == 0 && real)  // no key at all
          for (int i = 0; i < U; i++) reinterpret_cast<uint4*>(p.out + out_row * D)[i] = make_uint4(0, 0, 0, 0);
        continue;
      }
      // the query: asynchronous copies in memory's order, then each thread scales its own row by a power of two
#pragma unroll 4
      for (int x = 0; x < U; x++) {
        const int from = x * kPass + lane / U;
        const int64_t at = __shfl_sync(0xffffffffu, q_at, from);
        ptx::cp_async16(unit(w0 + from, lane % U), p.q + max(at, (int64_t)0) + 8 * (lane % U), at >= 0);
      }
      ptx::cp_async_wait_all();
      __syncwarp();
      float cq;
      {
        __nv_bfloat162 mx = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < U; k++) {
          const uint4 qv = *unit(r, k);
          const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&qv);
#pragma unroll
          for (int e = 0; e < 4; e++) mx = __hmax2(mx, __habs2(h[e]));
        }
        const float2 m2 = __bfloat1622float2(mx);
        const int qe = pre_exponent(__float_as_uint(fmaxf(m2.x, m2.y)));
        const float qf = pre_pow2(kTop - qe);
#pragma unroll 2
        for (int k = 0; k < U; k++) {
          float f[8];
          unpack8(*unit(r, k), f);
          uint32_t h[4];
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const __half2 y = __floats2half2_rn(f[2 * x] * qf, f[2 * x + 1] * qf);
            h[x] = *reinterpret_cast<const uint32_t*>(&y);
          }
          *unit(r, k) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        cq = p.scale_log2 * pre_pow2(qe - kTop);
      }
      ptx::fence_proxy_async();
      ptx::mbar_arrive(&q_full[t]);

      // the running maximum in the log2 domain, the sum, and the exponent that O's values of V stand under
      float m = -INFINITY, l = 0.f;
      int vrun = -100;
      for (int j = j0; j < j1; j++, n++) {
        ok = __all_sync(0xffffffffu, wait_for(&s_full[t], n & 1));
        if (!ok) break;
        ptx::tc_fence_after();
        const float c = cq * pre_pow2(s_exp[n & 3][0] - kTop);
        const int ve = s_exp[n & 3][1];
        uint32_t v[128];
#pragma unroll
        for (int q = 0; q < 4; q++) ptx::tmem_ld32(s_t + q * 32, v + q * 32);
        ptx::tmem_wait_ld();
        const int key0 = j * kKeys;
        if (__any_sync(0xffffffffu, key0 + kKeys - 1 > pos)) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int seen = max(0, min(32, pos + 1 - key0 - 32 * q));  // of these 32 keys
            const uint32_t hide = seen < 32 ? 0xFFFFFFFFu << seen : 0u;
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (hide & (1u << i)) v[32 * q + i] = 0xFF800000u;  // -infinity
          }
        }
        float mx[4];
#pragma unroll
        for (int q = 0; q < 4; q++) mx[q] = __uint_as_float(v[q]);
#pragma unroll
        for (int i = 4; i < 128; i += 8)
#pragma unroll
          for (int q = 0; q < 4; q++)
            mx[q] = i + 4 < 128 ? fmaxf(fmaxf(mx[q], __uint_as_float(v[i + q])), __uint_as_float(v[min(i + 4 + q, 127)]))
                                : fmaxf(mx[q], __uint_as_float(v[i + q]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        if (__any_sync(0xffffffffu, j == j0 || top > m + kPreSlack || ve > vrun)) {
          const float mn = fmaxf(m, top);
          const float a = m == -INFINITY ? 0.f : ex2(m - mn);
          const int vn = max(vrun, ve);
          m = mn;
          l *= a;
          if (j > j0) {
            const float f = a * pre_pow2(max(-126, vrun - vn));
#pragma unroll 1
            for (int q = 0; q < D / 16; q++) {
              uint32_t o[16];
              ptx::tmem_ld16u(o_t + q * 16, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              ptx::tmem_st16(o_t + q * 16, o);
            }
          }
          vrun = vn;
        }
        // P times 2^(kPreBits + ve - vrun), back over the columns of S, and the row's sum
        const float add = kPreBits + (float)(ve - vrun);
        const float mc = (m == -INFINITY ? 0.f : -m) + add;
        const uint64_t cc = ptx::pair_f32(c, c), mm = ptx::pair_f32(mc, mc);
        uint64_t sum[2];
        sum[0] = sum[1] = ptx::pair_f32(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float x = __uint_as_float(v[q * 32 + 2 * i]), y = __uint_as_float(v[q * 32 + 2 * i + 1]);
            const float2 e = ptx::unpair_f32(ptx::fma_f32x2(ptx::pair_f32(x, y), cc, mm));
            const float a = ex2(e.x), b = ex2(e.y);
            sum[i & 1] = ptx::add_f32x2(sum[i & 1], ptx::pair_f32(a, b));
            const __half2 h = __floats2half2_rn(a, b);
            pk[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          ptx::tmem_st16(s_t + q * 16, pk);
          if (q + 1 == kFirst) {
            ptx::tmem_wait_st();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&p_part[t]);
          }
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        ptx::mbar_arrive(&p_full[t]);
        const float2 both = ptx::unpair_f32(ptx::add_f32x2(sum[0], sum[1]));
        l = fmaf(both.x + both.y, ex2(-add), l);
      }
      if (ok) ok = __all_sync(0xffffffffu, wait_for(&o_full[t], items & 1));
      if (!ok) break;
      // (read here: ahead of the wait it costs 1,000 cycles an item, 16 prompts 125 us)
      const bool hole0 = pos >= s_nan[items & 3][0], hole1 = pos >= s_nan[items & 3][NG - 1];
      items++;
      ptx::tc_fence_after();
      // the output: through this warp's rows of the query tile (read by no MMA any more), so that a store
      // covers whole rows; a split's in fp32, 32 channels at a time (a thread its own row straight to memory, 32 lines
      // an instruction: 113 instead of 105 us for 509 rows on 0-40K keys)
      const float unit_o = pre_pow2(vrun - kTop - (int)kPreBits);
      // no visible key: zeros; keys whose scores are all -infinity: NaN
      const bool none = l == 0.f && pos < j0 * kKeys;
      l = l == 0.f && !none ? NAN : l;
      const float scale_o = ns > 1 ? unit_o : none ? 0.f : unit_o / l;
      // a row that sees a V of NaN, by halves of the channels
      const float scale0 = hole0 ? NAN : scale_o, scale1 = hole1 ? NAN : scale_o;
      if (ns == 1) {
#pragma unroll 1
        for (int q = 0; q < D / 32; q++) {
          uint32_t v[32];
          ptx::tmem_ld32(o_t + q * 32, v);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int u = 0; u < 4; u++) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = none ? 0.f : __uint_as_float(v[u * 8 + i]) * (q < D / 64 ? scale0 : scale1);
            *unit(r, q * 4 + u) = pack8(f);
          }
        }
        __syncwarp();
#pragma unroll 4
        for (int x = 0; x < U; x++) {
          const int from = x * kPass + lane / U;
          const int64_t at = __shfl_sync(0xffffffffu, out_row, from);
          const uint4 y = *unit(w0 + from, lane % U);
          if (at >= 0) reinterpret_cast<uint4*>(p.out + at * D)[lane % U] = y;
        }
        __syncwarp();
      } else {
#pragma unroll 1
        for (int q = 0; q < D / 32; q++) {
          uint32_t v[32];
          ptx::tmem_ld32(o_t + q * 32, v);
          ptx::tmem_wait_ld();
          const float scale_q = q < D / 64 ? scale0 : scale1;
          auto cell = [&](int x, int k) {  // 16-byte unit k of row x, 128 bytes a row
            return reinterpret_cast<float4*>(rows_s + x * 128 + ((k ^ (x & 7)) << 4));
          };
#pragma unroll
          for (int u = 0; u < 8; u++) {
            float4 f;
            f.x = __uint_as_float(v[4 * u]) * scale_q, f.y = __uint_as_float(v[4 * u + 1]) * scale_q;
            f.z = __uint_as_float(v[4 * u + 2]) * scale_q, f.w = __uint_as_float(v[4 * u + 3]) * scale_q;
            *cell(r, u) = f;
          }
          __syncwarp();
#pragma unroll 4
          for (int x = 0; x < 8; x++) {
            const int from = x * 4 + lane / 8;
            const int to = __shfl_sync(0xffffffffu, real ? part : -1, from);
            const float4 y = *cell(w0 + from, lane & 7);
            if (to >= 0) reinterpret_cast<float4*>(p.part_o + (int64_t)to * D + q * 32)[lane & 7] = y;
          }
          __syncwarp();
        }
      }
      if (real && ns > 1) reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(m, l);
      ptx::tc_fence_before();
    }
    if (!ok) s_fail = 1;
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 12) ptx::tmem_dealloc(tmem, kTmem);
  if (threadIdx.x == 0 && s_fail && p.status) atomicExch(p.status, (int)kTimeout);
}

// Rows cut along their keys: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in order. A warp per
// (row, query head).
template <int D>
__global__ void __launch_bounds__(128) prefill_merge_kernel(PreParams p) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch();
  const int64_t rh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (rh >= (int64_t)p.T * p.hq) return;
  const uint2 of = p.part_at[rh / p.hq];
  const int ns = of.x & 0xFFFF, per = of.x >> 16;
  if (ns <= 1) return;
  const int64_t part = (int64_t)of.y * p.hq + rh % p.hq * per;
  const float* ml = p.part_ml + part * 2;
  float mx = -INFINITY;
  for (int i = lane; i < ns; i += 32) mx = fmaxf(mx, ml[2 * i]);
  mx = warp_max(mx);
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.f;
  const float* po = p.part_o + part * D + E * lane;  // a lane E neighbouring channels
#pragma unroll 4
  for (int i = 0; i < ns; i++) {
    const float2 t = reinterpret_cast<const float2*>(ml)[i];
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
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no visible key in any split: zeros
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<__nv_bfloat162*>(p.out + rh * D + E * lane + e) =
        __floats2bfloat162_rn(inv == 0.f ? 0.f : acc[e] * inv, inv == 0.f ? 0.f : acc[e + 1] * inv);
}

template <int D, int NG, int BS>
cudaError_t launch_prefill(const PreParams& p, int grid, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = once_per_device(configured, [] {
    return cudaFuncSetAttribute(prefill_kernel<D, NG, BS>, cudaFuncAttributeMaxDynamicSharedMemorySize, PreCfg<D>::kSmem);
  });
  if (e != cudaSuccess) return e;
  e = launch_ex(prefill_kernel<D, NG, BS>, dim3(grid), dim3(kPreThreads), PreCfg<D>::kSmem, stream, 0, p);
  if (e != cudaSuccess || p.parts == 0) return e;
  return launch_ex(prefill_merge_kernel<D>, dim3((unsigned)(((int64_t)p.T * p.hq + 3) / 4)), dim3(128), 0, stream, 0, p);
}

}  // namespace kv4

int64_t kv4_prefill_parts(int64_t T, int64_t S, int64_t hq, int64_t hkv, int64_t max_len, const int64_t* rows,
                          const int64_t* ctx) {
  if (T <= 0 || S <= 0 || hkv <= 0 || hq < hkv || hq / hkv > kv4::kRows) return 0;
  const int64_t tt2 = 2 * (kv4::kRows / (hq / hkv));
  const auto tiles_of = [&](int64_t r) { return (int)std::min<int64_t>((r + tt2 - 1) / tt2, 128); };
  const auto keys_of = [](int64_t n) { return (int)((std::min<int64_t>(n, INT32_MAX - kv4::kKeys) + kv4::kKeys - 1) / kv4::kKeys); };
  // splits of a sequence of t row tiles and any context up to that of k key tiles
  const auto splits = [&](int t, int k) {
    const int64_t items = t * hkv;
    return items >= 128 ? 1 : (int64_t)std::min((k + kv4::least_chunk(items) - 1) / kv4::least_chunk(items), kv4::most_splits(items));
  };
  if (rows != nullptr) {
    int64_t sum = 0;
    for (int64_t s = 0; s < S; s++) {
      if (rows[s] <= 0 || ctx[s] <= 0) continue;
      const int64_t n = tiles_of(rows[s]) * hkv >= 128 ? 1 : kv4::cut_of(tiles_of(rows[s]), (int)hkv, keys_of(ctx[s])).splits;
      if (n > 1) sum += rows[s] * n;
    }
    return sum;
  }
  const int k = keys_of(max_len);
  if (S == 1) return splits(tiles_of(T), k) > 1 ? T * splits(tiles_of(T), k) : 0;  // its rows are the step's
  // each sequence may be of the length that takes the most, and each row of the one that is cut the most
  int64_t seq = 0, row = 0;
  for (int t = 1; t <= tiles_of(T) && t * hkv < 128; t++) {
    const int64_t n = splits(t, k);
    if (n > 1) seq = std::max(seq, t * tt2 * n), row = std::max(row, n);
  }
  return std::min(S * seq, T * row);
}

cudaError_t launch_kv4_prefill(const Kv4PrefillArgs& a, cudaStream_t stream) {
  if (a.T == 0) return cudaSuccess;
  if (a.S == 0) return cudaMemsetAsync(a.out, 0, (size_t)a.T * a.hq * a.c.d * sizeof(__nv_bfloat16), stream);
  if (a.c.hkv <= 0 || a.hq % a.c.hkv != 0 || a.hq / a.c.hkv > kv4::kRows || a.parts < 0 || !(a.scale > 0.f))
    return cudaErrorInvalidValue;
  if (a.c.s_block >> 4 > UINT32_MAX || a.parts * a.hq > INT32_MAX) return cudaErrorInvalidValue;
  if (a.T > INT32_MAX / 2 || a.bt_cols * a.c.block_size > INT32_MAX - kv4::kKeys || a.T * a.hq > ((int64_t)1 << 32))
    return cudaErrorInvalidValue;
  kv4::PreParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_stride = a.q_stride;
  p.cache = static_cast<const uint8_t*>(a.c.base);
  p.s_block = a.c.s_block;
  p.num_blocks = a.c.num_blocks;
  p.block_tables = a.block_tables;
  p.bt_stride = a.bt_stride;
  p.bt_cols = (int)a.bt_cols;
  p.ctx_lens = a.ctx_lens;
  p.last_rows = a.last_rows;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.part_at = a.parts > 0 ? static_cast<uint2*>(a.part_at) : nullptr;
  p.next = a.next;
  p.status = a.status;
  p.T = (int)a.T;
  p.S = (int)a.S;
  p.hq = a.hq;
  p.hkv = a.c.hkv;
  p.G = a.hq / a.c.hkv;
  p.tt = kv4::kRows / p.G;
  p.parts = (int)a.parts;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  // items: at most a row tile per 2 tt rows and sequence, each times heads, and more where some are cut
  const int64_t most = (a.T / (2 * p.tt) + a.S) * p.hkv;
  const int grid = (int)(a.parts == 0 && most < a.num_sms ? most : a.num_sms);
  const cudaError_t e = cudaMemsetAsync(a.next, 0, sizeof(unsigned), stream);
  if (e != cudaSuccess) return e;
  return kv4::pick(a.c.d, a.c.groups, a.c.block_size, [&](auto d, auto ng, auto bs) {
    return kv4::launch_prefill<d, ng, bs>(p, grid, stream);
  });
}

}  // namespace es
