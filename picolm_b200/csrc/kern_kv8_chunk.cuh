// kern_kv8_chunk.cuh -- causal attention of several tokens a slot over the
// 8-bit paged cache, on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// Bound by the softmax (its exponentials and the work around them) and, for
// FP32 and FP16 activations, by the tensor pipe, which then runs every product
// twice (high part and residual).
//
// Work.  A query item is up to two 128-row tiles ("slots" A and B) of one
// entry and KV head: row r of a slot is token r / G, query head r % G of the
// G heads that share the KV head, so a few tokens already fill a tile and
// both slots read the same K/V tiles.  The K/V tiles of all items, in order,
// form one list in which every item starts with kItemCost empty places
// (what its start and end cost, in tiles), and every block (one per SM)
// takes an equal contiguous slice of it: long prompts balance by themselves,
// and few tokens over a long context are split along it.  The part of an
// item in a slice is a segment; an item over several blocks leaves one
// partial (m, l, o) a block in the workspace, and the block that leaves the
// last one merges them in the order of the blocks.
//
// Roles (512 threads = four warpgroups):
//   warps 0-3, 4-7   softmax of slots A, B: rotate, scale and split the
//                    slot's rows of q into shared memory; then thread r owns
//                    query row r = TMEM lane r and per tile turns its S into
//                    weights
//   warps 8-11       converters: codes to FP16 -- every code is exact -- in
//                    swizzled K and V tiles
//   warps 12, 13     MMA issuers of slots A, B (12 allocates TMEM)
//   warp 14          scheduler: publishes the slice's segments, up to four ahead
//   warp 15          loader: bulk copies of codes and scales from the pages
//                    into a ring, tiles ahead of the converters
// Per tile n the issuer of slot x issues S(n) = Q K^T and then O += P(n-1) V,
// so a slot's softmax overlaps its own next scores and the other slot's
// products.  Tiles are 64 rows: at head_dim 128 TMEM has no room for wider S
// beside P, and with P in S's place a slot's softmax and products follow one
// another (585 -> 960 us for 4 x 1024 tokens behind 8192 rows).  The code of
// a tile is kept short: unrolled over 128 columns, two slots at different
// places of it waited for instructions four cycles in five.
//
// Measured on one B200: a prompt of 2048 FP32 tokens, 32/4 heads of 64: 92 us
// (17 GFLOP, 187 TFLOP/s; the tensor pipe, which does it twice, is active
// 18% of the time, issue slots 45%); 4 chunks of up to 1024 BF16 tokens
// behind up to 8192 rows, 32/8 heads of 128: 460 us (684 TFLOP/s, 32%, 50%).
// A pair of tiles takes 1.5 to 1.8 us, of which 2^x alone would take 0.55;
// the start and the end of an item another 7 to 9 pairs' time.
//
// Scales and ranges.  K's scale multiplies 16 columns of S before the row
// maximum; V's goes into the weight, relative to a reference of the row (of
// the blocks that it sees) that is raised (with O rescaled) when a scale
// outgrows it fourfold, as the running maximum is when a score outgrows it by
// 2^8, so weights stay below 2^14.
// q is scaled by a power of two a row.  FP32 and FP16 activations (PARTS 2): q and
// the weights are FP16 high part + residual, and every few tiles O is added
// to sums with one rounded FP32 operation and starts from zero again: the
// tensor core truncates as it accumulates, which alone put the output off by
// 1.6e-8 for each 16 rows, always towards zero.
// BF16 ones (PARTS 1): q and the weights are rounded to FP16 once, at most
// 2^-11 relative, an eighth of what rounding the output to BF16 costs.  FP16
// ones too would be off by 1.7 times the rounding of their output.
#pragma once
#include <cstdint>
#include <cuda.h>

#include <type_traits>

#include "kern_kv8_attn.cuh"

namespace pl {

constexpr int kChRows = 128;       // query rows of a slot
constexpr int kChThreads = 512;
constexpr int kChLaunchRegs = 128;
constexpr int kChSoftmaxRegs = 184;
constexpr int kChConvertRegs = 72;
constexpr int kChOtherRegs = 72;
static_assert(256 * kChSoftmaxRegs + 128 * kChConvertRegs + 128 * kChOtherRegs <=
                  kChThreads * kChLaunchRegs,
              "register split exceeds the launch allocation");
constexpr int kChQueue = 4;            // segments between the scheduler and the others
constexpr float kChBase = 16.f;        // weight of a row's maximum under the largest scale
constexpr float kChRescaleLog2 = 8.f;  // raise the running maximum only past 2^8
constexpr float kChRefGrowth = 4.f;    // raise the scale reference only past 4x

// FP16 parts of q and of the weights.
template <typename T>
constexpr int ch_parts() {
  return std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
}

template <int HD, int PARTS>
struct ChShape {
  static constexpr int kBN = 64;                   // rows of a K/V tile: a page
  static constexpr int kHalves = HD / 64;          // 64-element (128-byte) halves of a row
  static constexpr int kQHalf = kChRows * 128;
  static constexpr int kQBytes = kQHalf * kHalves;
  static constexpr int kKVHalf = kBN * 128;
  static constexpr int kKVBytes = kKVHalf * kHalves;
  static constexpr int kKStages = HD == 64 ? 3 : 2;
  static constexpr int kVStages = HD == 64 ? 3 : PARTS == 2 ? 1 : 2;
  static constexpr int kRawBytes = kBN * HD;       // codes of a K or V tile
  static constexpr int kRaw = HD == 64 ? 8 : PARTS == 2 ? 2 : 4;  // ring of them
  static constexpr int kBlocks = kBN / kBlock;     // scales of a K or V tile
  // TMEM columns: S_A, S_B (kBN FP32 each), O_A, O_B (HD), P_A, P_B (kBN / 2 a
  // part), and at head_dim 64 with PARTS 2 the sums of O_A and O_B (HD)
  static constexpr int kPCols = kBN / 2 * PARTS;
  static __device__ __forceinline__ uint32_t col_s(int x) { return x * kBN; }
  static __device__ __forceinline__ uint32_t col_o(int x) { return 2 * kBN + x * HD; }
  static __device__ __forceinline__ uint32_t col_p(int x) {
    return 2 * kBN + 2 * HD + x * kPCols;
  }
  // PARTS 2: tiles between moves of O into its sums: 256 rows where the sums
  // have TMEM columns, 512 where they are in the workspace
  static constexpr bool kSumsInTmem = HD == 64;
  static constexpr int kFlushTiles = HD == 64 ? 4 : 8;
  static __device__ __forceinline__ uint32_t col_sum(int x) {
    return 2 * kBN + 2 * HD + 2 * kPCols + x * HD;
  }
  static_assert(2 * kBN + 2 * HD + 2 * kPCols + (kSumsInTmem && PARTS == 2 ? 2 * HD : 0) <= 512,
                "TMEM columns");
  // Places of the list before an item's tiles: what its start (rows of q) and
  // end (O, a merge) take, in tiles; more where the rows are longer.  Measured
  // in the types named, used for all.  1 x 2048
  // tokens / 4 x 1024 behind 8192 rows / 16 x 64 behind 1024, in us, at
  // head_dim 64 in FP32: 106, 518, 59 with 3; 98, 502, 55 with 7; 104, 502,
  // 53 with 12.  At head_dim 128 in BF16: 121, 477, 70 with 3; 107, 465, 61
  // with 7; 104, 461, 61 with 9; 107, 461, 61 with 12.
  static constexpr int kItemCost = HD == 64 ? 7 : 9;
  static constexpr int kMinPlaces = kItemCost + 1;  // of a block's slice, at least
  static constexpr int kPartFloats = 2 * kChRows * (HD + 2);  // a partial: [slot][o.., m, l][row]
};

// A segment, as the scheduler publishes it (tiles == 0: no more).
struct ChSeg {
  int slot, len, n_tok, tok0;  // of the entry
  int h, first;                // KV head; first token of the item
  int j0, j1, tiles;           // tiles of the segment; of the item
  int f0, parts;               // first block of the item, blocks that have a part
};

template <int HD, int PARTS>
struct ChSmem {
  using Sh = ChShape<HD, PARTS>;
  // 1024-byte aligned tiles (128-byte swizzle)
  uint8_t q[2][PARTS][Sh::kQBytes];
  uint8_t k[Sh::kKStages][Sh::kKVBytes];
  uint8_t v[Sh::kVStages][Sh::kKVBytes];
  uint8_t raw[Sh::kRaw][Sh::kRawBytes];
  float raw_scale[Sh::kRaw][2][kBlocksPerPage];  // of K and V, beside K's codes
  float scale[8][2][Sh::kBlocks];  // of tile n in n % 8, K and V
  uint32_t bad[8];                 // blocks of it with a scale that is not finite
  float2 base[8][HD / 2];          // a softmax warp's cosines of its slot's first position
  float2 step[24][HD / 2];         // of 0..7 and of 0, 8, .. 120 tokens further
  float q_scale[2][kChRows];
  double half_turns[HD / 2];
  long long prefix[kPlanSeqs + 1];
  ChSeg seg[kChQueue];
  uint64_t seg_full[kChQueue], seg_empty[kChQueue];
  uint64_t raw_full[Sh::kRaw], raw_empty[Sh::kRaw];
  uint64_t k_full[Sh::kKStages], k_empty[Sh::kKStages];
  uint64_t v_full[Sh::kVStages], v_empty[Sh::kVStages];
  uint64_t q_full[2], s_full[2], s_free[2], p_full[2][2], pv_done[2][2], mma_done[2];
  // the scales of tile n: eight deep, so that tile n + 8 follows softmax n
  uint64_t scale_full[8];
  uint64_t part_full, merge_full;
  long long warp_sum[kChThreads / 32];
  uint32_t tmem_base;
  int merge;
};

struct Kv8ChunkArgs {
  Kv8AttnArgs a;
  float* part;   // [2 * blocks][kPartFloats]
  float* sums;   // [blocks][2][HD][kChRows], PARTS 2: what O was moved out to
  int* arrived;  // [blocks], zero at rest: by the block where an item starts
};

// K/V tiles of the query item that starts at token `first` of an entry (at
// least one, which may be all masked: rows with nothing to attend are
// written too).
template <int BN>
__device__ __forceinline__ int ch_tiles(int len, int n_tok, int first, int per_item) {
  const int last = len - n_tok + min(n_tok, first + per_item) - 1;
  return last < 0 ? 1 : last / BN + 1;
}

__device__ __forceinline__ float2 turn(float2 a, float2 b) {
  return make_float2(a.x * b.x - a.y * b.y, a.y * b.x + a.x * b.y);
}

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kChThreads, 1) kv8_chunk_kernel(
    const __grid_constant__ Kv8ChunkArgs ca) {
  constexpr int PARTS = ch_parts<T>();
  using Sh = ChShape<HD, PARTS>;
  constexpr int BN = Sh::kBN, KS = Sh::kKStages, VS = Sh::kVStages, RS = Sh::kRaw;
  extern __shared__ uint8_t smem_raw[];
  ChSmem<HD, PARTS>& sm = *reinterpret_cast<ChSmem<HD, PARTS>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const Kv8AttnArgs& a = ca.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = a.g.n_kv_heads, G = a.group;
  const int slot_tok = kChRows / G, per_item = 2 * slot_tok;
  const uint32_t inv_g = (65536 + G - 1) / G;  // r / G = r * inv_g >> 16 for a slot's rows
  // Place of pair i in a table of cosines: the pairs that the lanes of a row
  // want at once (every fourth or eighth) lie side by side.
  const int pair_log = a.rope.type == PL_ROPE_LLAMA ? 2 : 3;
  auto place = [&](int i) {
    return (i & ((1 << pair_log) - 1)) * ((HD / 2) >> pair_log) + (i >> pair_log);
  };
  uint32_t* err = &a.g.head->err;

  if (tid < HD / 2) sm.half_turns[tid] = a.rope.half_turns[tid];
  if (tid == 0) {
    for (int s = 0; s < kChQueue; ++s) {
      mbar_init(&sm.seg_full[s], 1);
      mbar_init(&sm.seg_empty[s], 15);  // 8 softmax, 4 converter warps, 2 issuers, loader
    }
    for (int s = 0; s < RS; ++s) {
      mbar_init(&sm.raw_full[s], 1);
      mbar_init(&sm.raw_empty[s], 4);
    }
    for (int s = 0; s < KS; ++s) {
      mbar_init(&sm.k_full[s], 4);
      mbar_init(&sm.k_empty[s], 2);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&sm.v_full[s], 4);
      mbar_init(&sm.v_empty[s], 2);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sm.q_full[x], 4);
      mbar_init(&sm.s_full[x], 1);
      mbar_init(&sm.s_free[x], 4);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sm.p_full[x][b], 4);
        mbar_init(&sm.pv_done[x][b], 1);
      }
      mbar_init(&sm.mma_done[x], 1);
    }
    for (int s = 0; s < 8; ++s) mbar_init(&sm.scale_full[s], 4);
    mbar_init(&sm.part_full, 8);
    mbar_init(&sm.merge_full, 1);
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  __syncthreads();  // half_turns
  for (int t = tid; t < 24 * (HD / 2); t += kChThreads) {
    const int w = t / (HD / 2), i = t % (HD / 2);
    sm.step[w][place(i)] = rope_cs_fast(sm.half_turns[i], 1.0, w < 8 ? w : 8 * (w - 8));
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- places of every entry, scanned
  for (int i = warp; i < a.n; i += kChThreads / 32) {
    Kv8Entry en;
    const bool ok = kv8_entry(a.g, i, a.total, a.max_tok, a.seqs, a.start, en);
    if (!ok && blockIdx.x == 0 && lane == 0) atomicOr(err, ERR_BAD_ARG);
    long long places = 0;
    if (ok)
      for (int f = lane * per_item; f < en.n_tok; f += 32 * per_item)
        places += Sh::kItemCost + ch_tiles<BN>(en.len, en.n_tok, f, per_item);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) places += __shfl_xor_sync(0xffffffffu, places, d);
    if (lane == 0) sm.prefix[i] = places * heads;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  {
    const int per = (a.n + kChThreads - 1) / kChThreads, i0 = tid * per;
    long long mine = 0;
    for (int i = i0; i < min(a.n, i0 + per); ++i) mine += sm.prefix[i];
    long long x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) sm.warp_sum[warp] = x;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < kChThreads / 32; ++w) {
      before += w < warp ? sm.warp_sum[w] : 0;
      all += sm.warp_sum[w];
    }
    long long run = before + x - mine;
    for (int i = i0; i < min(a.n, i0 + per); ++i) {
      const long long u = sm.prefix[i];
      sm.prefix[i] = run;
      run += u;
    }
    if (tid == 0) sm.prefix[a.n] = all;
    __syncthreads();
  }
  const uint32_t tmem = sm.tmem_base;

  // The k-th published segment stays in its place until every role has
  // released it: a copy of it would cost each thread a dozen registers.  False
  // after the last one, and when none came in time, which is recorded.
  auto taken = [&](int k, bool there) -> bool {
    if (!there) atomicOr(err, ERR_TIMEOUT_EMPTY);
    return there && sm.seg[k % kChQueue].tiles > 0;
  };
  auto take = [&](int k) -> bool {  // by a whole warp
    return taken(k, mbar_wait_warp(&sm.seg_full[k % kChQueue], (k / kChQueue) & 1));
  };
  auto take_alone = [&](int k) -> bool {  // by one lane of its warp
    return taken(k, mbar_wait_short(&sm.seg_full[k % kChQueue], (k / kChQueue) & 1));
  };

  if (warp >= 12) {
    regs_dec<kChOtherRegs>();
    if (warp == 14) {
      // --------------------------------------------------------- scheduler
      if (lane == 0) {
        const long long total = sm.prefix[a.n];
        const long long most = (total + Sh::kMinPlaces - 1) / Sh::kMinPlaces;
        const long long blocks = most < gridDim.x ? most : gridDim.x;
        const int blk = blockIdx.x;
        auto block_of = [&](long long p) {
          return static_cast<int>(((p + 1) * blocks - 1) / total);
        };
        int k = 0;
        if (blk < blocks) {
          long long p = blk * total / blocks;
          const long long end = (blk + 1) * total / blocks;
          int i = 0, hi = a.n - 1;
          while (i < hi) {
            const int mid = (i + hi) >> 1;
            if (sm.prefix[mid + 1] > p) hi = mid; else i = mid + 1;
          }
          Kv8Entry en;
          kv8_entry(a.g, i, a.total, a.max_tok, a.seqs, a.start, en);
          const long long per_head = (sm.prefix[i + 1] - sm.prefix[i]) / heads;
          long long at = sm.prefix[i];  // the current item's first place
          int h = static_cast<int>((p - at) / per_head), first = 0;
          at += h * per_head;
          int tiles = ch_tiles<BN>(en.len, en.n_tok, 0, per_item);
          while (p >= at + Sh::kItemCost + tiles) {
            at += Sh::kItemCost + tiles;
            first += per_item;
            tiles = ch_tiles<BN>(en.len, en.n_tok, first, per_item);
          }
          while (true) {
            const long long t0 = at + Sh::kItemCost;  // place of the item's first tile
            ChSeg g;
            g.j0 = p > t0 ? static_cast<int>(p - t0) : 0;
            g.j1 = end - t0 < tiles ? static_cast<int>(end - t0) : tiles;
            if (g.j1 > g.j0) {
              g.slot = en.slot, g.len = en.len, g.n_tok = en.n_tok, g.tok0 = en.tok0;
              g.h = h, g.first = first, g.tiles = tiles;
              g.f0 = block_of(t0);
              g.parts = block_of(t0 + tiles - 1) - g.f0 + 1;
              if (k >= kChQueue &&
                  !mbar_wait_short(&sm.seg_empty[k % kChQueue], (k / kChQueue - 1) & 1)) {
                atomicOr(err, ERR_TIMEOUT_EMPTY);
                break;  // the others give up on their own waits
              }
              sm.seg[k % kChQueue] = g;
              mbar_arrive(&sm.seg_full[k % kChQueue]);
              ++k;
            }
            at = t0 + tiles;
            p = at;
            if (p >= end) break;
            first += per_item;
            if (first >= en.n_tok) {
              first = 0;
              if (++h == heads) {
                h = 0;
                do ++i; while (i < a.n && sm.prefix[i + 1] == sm.prefix[i]);
                if (i >= a.n) break;
                kv8_entry(a.g, i, a.total, a.max_tok, a.seqs, a.start, en);
              }
            }
            tiles = ch_tiles<BN>(en.len, en.n_tok, first, per_item);
          }
        }
        if (k < kChQueue ||
            mbar_wait_short(&sm.seg_empty[k % kChQueue], (k / kChQueue - 1) & 1)) {
          sm.seg[k % kChQueue].tiles = 0;
          mbar_arrive(&sm.seg_full[k % kChQueue]);
        }
      }
    } else if (warp == 15) {
      // ------------------------------------------------------------ loader
      int u = 0;  // K or V tiles loaded
      bool ok = true;
      for (int k = 0; ok && take(k); ++k) {
        const ChSeg& g = sm.seg[k % kChQueue];
        const int nt = g.j1 - g.j0;
        const int* row = a.g.table + static_cast<long long>(g.slot) * a.g.max_pages;
        const int pages = (g.len + kPage - 1) / kPage;
        int mine = 0, batch = -64;  // lane's page of the batch of 32
        // K of tile n + 1 goes before V of tile n
        for (int w = 0; w < 2 * nt && ok; ++w, ++u) {
          const bool is_v = w == 2 * nt - 1 || (w > 0 && !(w & 1));
          const int n = is_v ? (w == 2 * nt - 1 ? nt - 1 : w / 2 - 1) : (w + 1) / 2;
          const int at = g.j0 + n;  // page of the sequence
          // V of a batch's last tile may follow K of the next one: it asks again
          if (at < batch || at >= batch + 32) {
            batch = at;
            mine = batch + lane < pages ? row[batch + lane] : 0;
            if (mine < 0 || mine >= a.g.n_pages) {
              atomicOr(err, ERR_BAD_ARG);
              mine = 0;
            }
          }
          const int page = __shfl_sync(0xffffffffu, mine, at - batch);
          const int s = u % RS;
          if (u >= RS && !mbar_wait_warp(&sm.raw_empty[s], ((u / RS) - 1) & 1)) {
            if (lane == 0) atomicOr(err, ERR_TIMEOUT_EMPTY);
            ok = false;
            break;
          }
          if (lane == 0) {
            // (a sequence with no row has one tile and no page)
            const bool have = at < pages;
            mbar_arrive_expect_tx(&sm.raw_full[s],
                                  have ? kPage * HD + (is_v ? 0 : 8 * kBlocksPerPage) : 0);
            if (have) {
              const long long slab = a.g.slab(page, g.h, is_v);
              bulk_load(sm.raw[s], a.g.codes + slab * kPage * HD, kPage * HD, &sm.raw_full[s]);
              if (!is_v)
                bulk_load(sm.raw_scale[s], a.g.scales + slab * kBlocksPerPage,
                          8 * kBlocksPerPage, &sm.raw_full[s]);
            }
          }
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&sm.seg_empty[k % kChQueue]);
      }
      // never leave with copies in flight
      for (int w = max(u - RS, 0); w < u; ++w)
        mbar_wait_drained(&sm.raw_full[w % RS], (w / RS) & 1);
    } else if (lane == 0) {
      // ------------------------------------------------- MMA issuer of slot x
      const int x = warp - 12;
      const uint32_t idesc_qk = idesc_f16_f32(128, BN, 0);
      const uint32_t idesc_pv = idesc_f16_f32(128, 64, 1);
      const uint32_t q_addr = smem_u32(sm.q[x][0]);
      int J = 0, A = 0, kq = 0;  // tiles of the block; tiles and segments of this slot
      bool ok = true;
      // O += P V of the block's tile n, the slot's tile m
      auto issue_pv = [&](int n, int m, bool fresh) -> bool {
        const int vs = n % VS;
        if (!mbar_wait_short(&sm.v_full[vs], (n / VS) & 1) ||
            !mbar_wait_short(&sm.p_full[x][m & 1], (m >> 1) & 1))
          return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sm.v[vs]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int hv = 0; hv < Sh::kHalves; ++hv)
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk) {
              const uint64_t bd =
                  smem_desc_sw128(v_addr + hv * Sh::kKVHalf + kk * 16 * 128, 16, 1024);
              tc_mma_ts(tmem + Sh::col_o(x) + 64 * hv,
                        tmem + Sh::col_p(x) + part * (BN / 2) + kk * 8, bd, idesc_pv,
                        (fresh && part == 0 && kk == 0) ? 0u : 1u);
            }
        tc_commit(&sm.pv_done[x][m & 1]);
        tc_commit(&sm.v_empty[vs]);
        return true;
      };
      for (int k = 0; ok && take_alone(k); ++k) {
        const ChSeg& g = sm.seg[k % kChQueue];
        const int nt = g.j1 - g.j0;
        const bool active = g.first + x * slot_tok < g.n_tok;
        if (active) {
          ok = mbar_wait_short(&sm.q_full[x], kq & 1);
          ++kq;
        }
        auto fresh = [&](int j) { return j == 0 || (PARTS == 2 && j % Sh::kFlushTiles == 0); };
        for (int j = 0; j < nt && ok; ++j) {
          const int n = J + j, ks = n % KS;
          if (!mbar_wait_short(&sm.k_full[ks], (n / KS) & 1)) { ok = false; break; }
          if (!active) {  // no token of the item in this slot: it only frees the tiles
            mbar_arrive(&sm.k_empty[ks]);
            if (!mbar_wait_short(&sm.v_full[n % VS], (n / VS) & 1)) { ok = false; break; }
            mbar_arrive(&sm.v_empty[n % VS]);
            continue;
          }
          if (A >= 1 && !mbar_wait_short(&sm.s_free[x], (A - 1) & 1)) { ok = false; break; }
          tc_fence_after();
          const uint32_t k_addr = smem_u32(sm.k[ks]);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off_q = (kk >> 2) * Sh::kQHalf + (kk & 3) * 32;
            const uint64_t bd =
                smem_desc_sw128(k_addr + (kk >> 2) * Sh::kKVHalf + (kk & 3) * 32, 16, 1024);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
              tc_mma_ss(tmem + Sh::col_s(x),
                        smem_desc_sw128(q_addr + part * Sh::kQBytes + off_q, 16, 1024), bd,
                        idesc_qk, kk + part > 0 ? 1u : 0u);
          }
          tc_commit(&sm.s_full[x]);
          tc_commit(&sm.k_empty[ks]);
          if (j >= 1 && !issue_pv(n - 1, A - 1, fresh(j - 1))) ok = false;
          ++A;
        }
        if (ok && active && !issue_pv(J + nt - 1, A - 1, fresh(nt - 1))) ok = false;
        J += nt;
        mbar_arrive(&sm.seg_empty[k % kChQueue]);
      }
      if (!ok) atomicOr(err, ERR_TIMEOUT_MMA);
      // all issued MMAs must finish before TMEM is freed
      tc_commit(&sm.mma_done[x]);
      mbar_wait_drained(&sm.mma_done[x], 0);
    }
  } else if (warp >= 8) {
    regs_dec<kChConvertRegs>();
    // ----------------------------------------------------------- converters
    const int pt = tid - 256;
    constexpr int kPerRow = HD / 16;  // 16-byte chunks of a row of codes
    const int ch = pt % kPerRow, row0 = pt / kPerRow;
    const uint32_t dst0 = (ch >> 2) * Sh::kKVHalf + row0 * 128;
    const uint32_t at0 = ((2 * (ch & 3)) ^ (row0 & 7)) << 4;
    int u = 0, J = 0;
    bool ok = true;
    for (int k = 0; ok && take(k); ++k) {
      const ChSeg& g = sm.seg[k % kChQueue];
      const int nt = g.j1 - g.j0;
      for (int w = 0; w < 2 * nt; ++w, ++u) {
        const bool is_v = w == 2 * nt - 1 || (w > 0 && !(w & 1));
        const int j = is_v ? (w == 2 * nt - 1 ? nt - 1 : w / 2 - 1) : (w + 1) / 2;
        const int n = J + j, rs = u % RS, stages = is_v ? VS : KS, s = n % stages;
        if (!__all_sync(0xffffffffu,
                        mbar_wait_short(&sm.raw_full[rs], (u / RS) & 1) &&
                            (n < stages || mbar_wait_short(is_v ? &sm.v_empty[s] : &sm.k_empty[s],
                                                           ((n / stages) - 1) & 1)))) {
          if (lane == 0) atomicOr(err, ERR_TIMEOUT_EMPTY);
          ok = false;
          break;
        }
        constexpr int kChunks = BN * kPerRow / 128, kRowStep = 128 / kPerRow;
        const uint4* src = reinterpret_cast<const uint4*>(sm.raw[rs]) + pt;
        uint8_t* dst = (is_v ? sm.v[s] : sm.k[s]) + dst0;
        const int left = g.len - (g.j0 + j) * BN;  // rows of the tile that exist
        uint4 in[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) in[c] = src[c * 128];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t w4[4] = {in[c].x, in[c].y, in[c].z, in[c].w};
          uint32_t o[8];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            o[2 * q] = codes_half2<FMT, 0x10>(w4[q]);
            o[2 * q + 1] = codes_half2<FMT, 0x32>(w4[q]);
          }
          // elements 16 ch ..: chunks 2ch, 2ch + 1 of a 64-element half; rows
          // are kRowStep (a multiple of 8) apart, so the swizzle is row0's
          *reinterpret_cast<uint4*>(dst + c * kRowStep * 128 + at0) =
              make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + c * kRowStep * 128 + (at0 ^ 16)) =
              make_uint4(o[4], o[5], o[6], o[7]);
        }
        if (left < BN) {  // rows past the end: anything was there, NaN codes too
#pragma unroll 1
          for (int row = row0, o = 0; row < BN; row += kRowStep, o += kRowStep * 128)
            if (row >= left) {
              *reinterpret_cast<uint4*>(dst + o + at0) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(dst + o + (at0 ^ 16)) = make_uint4(0, 0, 0, 0);
            }
        }
        if (!is_v && pt < 32) {
          // A scale that is not finite becomes 0 and leaves a bit: rows that see
          // its block are made NaN, and 0 times what a mask hides stays 0 (the
          // codes of rows that exist are never NaN).
          const int kv = pt / Sh::kBlocks & 1, b = pt % Sh::kBlocks;
          const float f = b * kBlock < left ? sm.raw_scale[rs][kv][b] : 0.f;
          const uint32_t odd =
              __ballot_sync(0xffffffffu, pt < 2 * Sh::kBlocks && !(f < INFINITY));
          if (pt < 2 * Sh::kBlocks) sm.scale[n & 7][kv][b] = f < INFINITY ? f : 0.f;
          if (pt == 0) sm.bad[n & 7] = (odd | odd >> Sh::kBlocks) & ((1u << Sh::kBlocks) - 1);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.raw_empty[rs]);
          mbar_arrive(is_v ? &sm.v_full[s] : &sm.k_full[s]);
          if (!is_v) mbar_arrive(&sm.scale_full[n & 7]);
        }
      }
      J += nt;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.seg_empty[k % kChQueue]);
    }
  } else {
    regs_inc<kChSoftmaxRegs>();
    // -------------------------------------------------------------- softmax
    const int x = warp >> 2;        // slot
    const int r = tid & 127;        // query row of the slot, TMEM lane
    const int row_tok = r * inv_g >> 16, row_head = r - row_tok * G;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int J = 0, A = 0, n_merge = 0;
    // a wait that gave up ends this warp's arithmetic; it still takes its
    // part in the barriers, each of which is bounded too
    bool ok = true;
    for (int k = 0; take(k); ++k) {
      const ChSeg& g = sm.seg[k % kChQueue];
      const int nt = g.j1 - g.j0;
      const int tok_x = g.first + x * slot_tok;  // the slot's first token
      const bool active = tok_x < g.n_tok;
      const bool whole = nt == g.tiles;
      const bool real = row_tok < slot_tok && tok_x + row_tok < g.n_tok;
      const int p_min = g.len - g.n_tok + tok_x;   // position of the slot's first token
      const int pos = real ? p_min + row_tok : -1;
      float m_used = -INFINITY, l_run = 0.f, ref = kMinRef, q_scale = 0.f;
      float unit = kChBase / kMinRef;  // what V's scales are multiplied by
      float m_sum = -INFINITY, ref_sum = kMinRef;  // of the sums outside TMEM
      const long long out_row = static_cast<long long>(g.tok0) + tok_x + row_tok;
      const int head_el = (g.h * G + row_head) * HD;
      float* sums = PARTS == 2 ? ca.sums + (static_cast<long long>(blockIdx.x) * 2 + x) * HD * kChRows + r
                               : nullptr;
      if (active && ok) {
        // ---- the warp's 32 rows of q: rotated, scaled, split, into the tile.
        // HD / 8 lanes share a row, so that loads are whole lines (a row a
        // thread took 11 us a segment at head_dim 128), eight loads at a time.
        constexpr int LR = HD / 8, RI = 32 / LR;  // lanes of a row, rows at once
        const int e = (lane % LR) * 8, half = a.rope.dim >> 1;
        const bool llama = a.rope.type == PL_ROPE_LLAMA;
        for (int i = lane; i < half; i += 32)
          sm.base[warp][place(i)] = rope_cs_fast(sm.half_turns[i], a.rope.gain, p_min);
        __syncwarp();
        auto row_at = [&](int it) { return (warp & 3) * 32 + it * RI + lane / LR; };
        const int n_tok = g.n_tok;
        const T* q_slot = static_cast<const T*>(a.q) +
                          (static_cast<long long>(g.tok0) + tok_x) * a.q_stride + g.h * G * HD;
        auto q_row = [&](int row, bool& there) -> const T* {
          const int tk = row * inv_g >> 16;
          there = tk < slot_tok && tok_x + tk < n_tok;
          if (!there) return static_cast<const T*>(a.q);
          return q_slot + tk * a.q_stride + (row - tk * G) * HD;
        };
        // four rows ahead; the loop is not unrolled, because it runs once a
        // segment and fetching the unrolled code took longer than running it
        Raw8<T> raw[4];
        bool there;
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[k] = raw8(q_row(row_at(k), there) + e);
        float2 f[8];  // cosines of this lane's elements at token cs_tok
        int cs_tok = -1;
#pragma unroll 1
        for (int it = 0; it < LR; ++it) {
          const int row = row_at(it), tk = row * inv_g >> 16;
          float y[8];
          unpack8(raw[0], y);
#pragma unroll
          for (int k = 0; k < 3; ++k) raw[k] = raw[k + 1];
          if (it + 4 < LR) raw[3] = raw8(q_row(row_at(it + 4), there) + e);
          const T* q = q_row(row, there);
          if (!there) {
#pragma unroll
            for (int d = 0; d < 8; ++d) y[d] = 0.f;
          }
          if (__any_sync(0xffffffffu, there && tk != cs_tok)) {
            cs_tok = tk;
            const int tt = min(tk, kChRows - 1);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const int el = e + d;
              if (llama && (d & 1)) continue;
              const int i = place(llama ? el >> 1 : el < half ? el : el - half);
              if (el < a.rope.dim)
                f[d] = turn(turn(sm.base[warp][i], sm.step[8 + (tt >> 3)][i]), sm.step[tt & 7][i]);
            }
          }
          if (llama) {
#pragma unroll
            for (int d = 0; d < 8; d += 2)
              if (e + d < a.rope.dim) {
                const float u = y[d], v = y[d + 1];
                y[d] = u * f[d].x - v * f[d].y;
                y[d + 1] = u * f[d].y + v * f[d].x;
              }
          } else {
            float o[8];  // the partners: in another lane, or in memory
            if (a.rope.dim == HD) {
#pragma unroll
              for (int d = 0; d < 8; ++d) o[d] = __shfl_xor_sync(0xffffffffu, y[d], LR / 2);
            } else {
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                const int el = e + d;
                o[d] = there && el < a.rope.dim ? to_f32(q[el < half ? el + half : el - half]) : 0.f;
              }
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
              if (e + d < a.rope.dim) {
                const float s = e + d < half ? -f[d].y : f[d].y;
                y[d] = fmaf(y[d], f[d].x, o[d] * s);
              }
          }
          float top = 0.f;
#pragma unroll
          for (int d = 0; d < 8; ++d) top = fmaxf(top, fabsf(y[d]));
#pragma unroll
          for (int o = 1; o < LR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const uint32_t ex = __float_as_uint(top) >> 23;
          const bool norm = ex > 1 && ex < 253;
          const float down = norm ? __uint_as_float((254u - ex) << 23) : 1.f;
          if (lane % LR == 0)
            sm.q_scale[x][row] = (norm ? __uint_as_float(ex << 23) : 1.f) * a.score_scale;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const float u = y[2 * d] * down, v = y[2 * d + 1] * down;
            if constexpr (PARTS == 2) split_hi_lo(u, v, hi[d], lo[d]);
            else hi[d] = pack_half2(u, v);
          }
          const uint32_t off =
              (e >> 6) * Sh::kQHalf + row * 128 + ((((e >> 3) & 7) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(sm.q[x][0] + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (PARTS == 2)
            *reinterpret_cast<uint4*>(sm.q[x][PARTS - 1] + off) =
                make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        __syncwarp();
        q_scale = sm.q_scale[x][r];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[x]);
      }
      // O, relative to (m_used, ref), joins its sums
      auto flush = [&](bool first) {
        const float ms = m_used == -INFINITY ? 0.f : m_used;
        const float old = first ? 0.f : ex2(m_sum - ms) * (ref_sum / ref);
#pragma unroll 1
        for (int d0 = 0; d0 < HD; d0 += 16) {
          uint32_t ov[16], sv[16] = {};
          tc_ld_32x32b_x16(lane_base + Sh::col_o(x) + d0, ov);
          if (!first) {
            if constexpr (Sh::kSumsInTmem) {
              tc_ld_32x32b_x16(lane_base + Sh::col_sum(x) + d0, sv);
            } else {
#pragma unroll
              for (int d = 0; d < 16; ++d) sv[d] = __float_as_uint(sums[(d0 + d) * kChRows]);
            }
          }
          tc_wait_ld();
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            asm volatile("" : "+r"(ov[d]), "+r"(sv[d]));
            sv[d] = __float_as_uint(fmaf(__uint_as_float(sv[d]), old, __uint_as_float(ov[d])));
          }
          if constexpr (Sh::kSumsInTmem) {
            tc_st_32x32b_x16(lane_base + Sh::col_sum(x) + d0, sv);
          } else {
#pragma unroll
            for (int d = 0; d < 16; ++d) sums[(d0 + d) * kChRows] = __uint_as_float(sv[d]);
          }
        }
        if constexpr (Sh::kSumsInTmem) tc_wait_st();
        m_sum = m_used;
        ref_sum = ref;
      };
      for (int j = 0; j < nt && active; ++j, ++A) {
        const int n = J + j;
        // (the scales are the converters' writes: their barriers too.  A slot
        // that sat out eight tiles or more can find the barrier two phases back
        // and pass early; s_full then orders the writes, since the issuer took
        // the same warps' k_full of this tile, arrived at after the scales.)
        ok = __all_sync(0xffffffffu, ok && mbar_wait_short(&sm.scale_full[n & 7], (n >> 3) & 1) &&
                                         mbar_wait_short(&sm.s_full[x], A & 1));
        if (!ok) continue;
        tc_fence_after();
        uint32_t u[BN];
#pragma unroll
        for (int q = 0; q < BN / 32; ++q)
          tc_ld_32x32b_x32(lane_base + Sh::col_s(x) + 32 * q,
                           *reinterpret_cast<uint32_t(*)[32]>(u + 32 * q));
        tc_wait_ld();
#pragma unroll
        for (int d = 0; d < BN; ++d) asm volatile("" : "+r"(u[d]));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_free[x]);
        const int t0 = (g.j0 + j) * BN;
        const bool need_mask = t0 + BN - 1 > p_min;
        const int lim = pos - t0;  // columns c <= lim are visible
        float sk[Sh::kBlocks], sv[Sh::kBlocks];
        {
          const float4 fk = *reinterpret_cast<const float4*>(sm.scale[n & 7][0]);
          const float4 fv = *reinterpret_cast<const float4*>(sm.scale[n & 7][1]);
          sk[0] = fk.x, sk[1] = fk.y, sk[2] = fk.z, sk[3] = fk.w;
          sv[0] = fv.x, sv[1] = fv.y, sv[2] = fv.z, sv[3] = fv.w;
        }
        // what a block's scores are multiplied by; never 0, which would make a
        // masked -inf NaN (the codes under a scale of 0 are 0)
#pragma unroll
        for (int b = 0; b < Sh::kBlocks; ++b) sk[b] = fmaxf(sk[b] * q_scale, 1e-30f);
        if (const uint32_t bad = sm.bad[n & 7]) {
          if (lim >= 16 * (__ffs(bad) - 1)) l_run = NAN;
        }
        if (need_mask) {
#pragma unroll
          for (int c = 0; c < BN; ++c) {
            if (c > lim) u[c] = __float_as_uint(-INFINITY);
            asm volatile("" : "+r"(u[c]));  // a branch, not 64 selects in every tile
          }
          // blocks that are hidden whole weigh nothing and leave the row's
          // reference where it is: later tokens' values do not reach this one
#pragma unroll
          for (int b = 0; b < Sh::kBlocks; ++b) {
            if (16 * b > lim) sv[b] = 0.f;
            asm volatile("" : "+f"(sv[b]));
          }
        }
        // ---- the row's maximum: of a block's columns, times its scale (which
        // is not negative), over the blocks
        float m_tile = -INFINITY;
#pragma unroll
        for (int b = 0; b < Sh::kBlocks; ++b) {
          auto at = [&](int c) { return __uint_as_float(u[16 * b + c]); };
          const float z = max3(max3(max3(at(0), at(1), at(2)), max3(at(3), at(4), at(5)),
                                    max3(at(6), at(7), at(8))),
                               max3(at(9), at(10), at(11)),
                               max3(max3(at(12), at(13), at(14)), at(15), at(15)));
          m_tile = fmaxf(m_tile, z * sk[b]);
        }
        const float top_v = max3(fmaxf(sv[0], sv[1]), sv[2], sv[3]);
        const bool rescale = __any_sync(
            0xffffffffu, m_tile > m_used + kChRescaleLog2 || top_v > kChRefGrowth * ref);
        const bool moved = PARTS == 2 && j > 0 && j % Sh::kFlushTiles == 0;
        // O and P are free to change once PV of the tile before is done (a lane's
        // verdict joins the others' at the warp's next vote)
        if (A >= 1 && !mbar_wait_short(&sm.pv_done[x][(A - 1) & 1], ((A - 1) >> 1) & 1))
          ok = false;
        tc_fence_after();
        if (moved) flush(j == Sh::kFlushTiles);
        if (rescale) {
          const float m_new = fmaxf(m_used, m_tile);
          const float alpha = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
          const float ref_new = fmaxf(ref, top_v);
          const float keep = alpha * (ref / ref_new);
          l_run *= alpha;
          m_used = m_new;
          ref = ref_new;
          unit = kChBase / ref;
          if (j > 0 && !moved) {
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += 16) {
              uint32_t ov[16];
              tc_ld_32x32b_x16(lane_base + Sh::col_o(x) + d0, ov);
              tc_wait_ld();
#pragma unroll
              for (int d = 0; d < 16; ++d) {
                asm volatile("" : "+r"(ov[d]));
                ov[d] = __float_as_uint(__uint_as_float(ov[d]) * keep);
              }
              tc_st_32x32b_x16(lane_base + Sh::col_o(x) + d0, ov);
            }
          }
        }
        const float m_safe = m_used == -INFINITY ? 0.f : m_used;
        const float2 nm2 = make_float2(-m_safe, -m_safe);
        float2 rs2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // ---- the weights, 32 columns at a time
#pragma unroll
        for (int q = 0; q < BN / 32; ++q) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int b = 2 * q; b < 2 * q + 2; ++b) {
            const float kb = sk[b], vb = sv[b] * unit;
#pragma unroll
            for (int e = 8 * b; e < 8 * b + 8; ++e) {
              const float2 arg =
                  fma2(make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1])),
                       make_float2(kb, kb), nm2);
              const float2 p = make_float2(ex2(arg.x), ex2(arg.y));
              rs2[e & 1] = add2(rs2[e & 1], p);
              const float2 w = mul2(p, make_float2(vb, vb));
              if constexpr (PARTS == 2) split_hi_lo(w.x, w.y, hi[e - 16 * q], lo[e - 16 * q]);
              else hi[e - 16 * q] = pack_half2(w.x, w.y);
            }
          }
          tc_st_32x32b_x16(lane_base + Sh::col_p(x) + 16 * q, hi);
          if constexpr (PARTS == 2)
            tc_st_32x32b_x16(lane_base + Sh::col_p(x) + BN / 2 + 16 * q, lo);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[x][A & 1]);
        const float2 ra = add2(rs2[0], rs2[1]);
        l_run += ra.x + ra.y;
      }
      J += nt;
      float* part = ca.part +
                    static_cast<long long>(2 * blockIdx.x + (g.j0 > 0 ? 0 : 1)) * Sh::kPartFloats +
                    x * kChRows * (HD + 2) + r;
      if (active) {
        // ---- the segment's O
        ok = __all_sync(0xffffffffu,
                        ok && mbar_wait_short(&sm.pv_done[x][(A - 1) & 1], ((A - 1) >> 1) & 1));
        tc_fence_after();
        if (ok) {
          const float back = ref * (1.f / kChBase);
          const float by = whole ? (l_run == 0.f ? 0.f : back / l_run) : back;
          const bool summed = PARTS == 2 && nt > Sh::kFlushTiles;
          const float ms = m_used == -INFINITY ? 0.f : m_used;
          const float old = summed ? ex2(m_sum - ms) * (ref_sum / ref) : 0.f;
#pragma unroll 1
          for (int d0 = 0; d0 < HD; d0 += 32) {
            uint32_t ov[32], su[32] = {};
            tc_ld_32x32b_x32(lane_base + Sh::col_o(x) + d0, ov);
            if (summed) {
              if constexpr (Sh::kSumsInTmem) {
                tc_ld_32x32b_x32(lane_base + Sh::col_sum(x) + d0, su);
              } else {
#pragma unroll
                for (int d = 0; d < 32; ++d) su[d] = __float_as_uint(sums[(d0 + d) * kChRows]);
              }
            }
            tc_wait_ld();
            float z[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) {
              asm volatile("" : "+r"(ov[d]), "+r"(su[d]));
              z[d] = fmaf(__uint_as_float(su[d]), old, __uint_as_float(ov[d])) * by;
            }
            if (!whole) {
#pragma unroll
              for (int d = 0; d < 32; ++d) part[(d0 + d) * kChRows] = z[d];
            } else if (real) {
              T* dst = static_cast<T*>(a.out) + out_row * a.out_stride + head_el + d0;
#pragma unroll
              for (int d = 0; d < 32; d += 8) store8(dst + d, *reinterpret_cast<float(*)[8]>(z + d));
            }
          }
          if (!whole) {
            part[HD * kChRows] = m_used;
            part[(HD + 1) * kChRows] = l_run;
          }
        }
        tc_fence_before();
      }
      if (!whole) {
        // ---- leave the partial; the last block of the item merges them
        __threadfence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.part_full);
        if (tid == 0) {
          const bool whole_part = mbar_wait_short(&sm.part_full, n_merge & 1);
          if (!whole_part) atomicOr(err, ERR_TIMEOUT_MMA);  // and it does not count
          const bool done = whole_part && atomicAdd(&ca.arrived[g.f0], 1) == g.parts - 1;
          if (done) ca.arrived[g.f0] = 0;
          sm.merge = done;
          __threadfence();
          mbar_arrive(&sm.merge_full);
        }
        __syncwarp();
        if (!mbar_wait_warp(&sm.merge_full, n_merge & 1)) ok = false;
        ++n_merge;
        if (*reinterpret_cast<volatile int*>(&sm.merge) && real && ok) {
          // the first block's partial is of kind 1, the others' of kind 0
          const float* p0 = ca.part + static_cast<long long>(2 * g.f0) * Sh::kPartFloats +
                            x * kChRows * (HD + 2) + r;
          auto at = [&](int p) {
            return p0 + static_cast<long long>(2 * p + (p == 0)) * Sh::kPartFloats;
          };
          float M = -INFINITY, L = 0.f;
          for (int p = 0; p < g.parts; ++p) M = fmaxf(M, __ldcg(at(p) + HD * kChRows));
          const float Ms = M == -INFINITY ? 0.f : M;
          for (int p = 0; p < g.parts; ++p)
            L += ex2(__ldcg(at(p) + HD * kChRows) - Ms) * __ldcg(at(p) + (HD + 1) * kChRows);
          const float inv = L == 0.f ? 0.f : 1.f / L;
          T* dst = static_cast<T*>(a.out) + out_row * a.out_stride + head_el;
#pragma unroll 1
          for (int d0 = 0; d0 < HD; d0 += 32) {
            float z[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) z[d] = 0.f;
#pragma unroll 1
            for (int p = 0; p < g.parts; p += 2) {  // 64 loads in flight
              const float *pa = at(p), *pb = at(min(p + 1, g.parts - 1));
              float u[32], v[32];
#pragma unroll
              for (int d = 0; d < 32; ++d) {
                u[d] = __ldcg(pa + (d0 + d) * kChRows);
                v[d] = __ldcg(pb + (d0 + d) * kChRows);
              }
              const float wa = ex2(__ldcg(pa + HD * kChRows) - Ms) * inv;
              const float wb =
                  p + 1 < g.parts ? ex2(__ldcg(pb + HD * kChRows) - Ms) * inv : 0.f;
#pragma unroll
              for (int d = 0; d < 32; ++d) z[d] = fmaf(wb, v[d], fmaf(wa, u[d], z[d]));
            }
#pragma unroll
            for (int d = 0; d < 32; d += 8)
              store8(dst + d0 + d, *reinterpret_cast<float(*)[8]>(z + d));
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.seg_empty[k % kChQueue]);
    }
    if (!ok) atomicOr(err, ERR_TIMEOUT_MMA);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace pl
