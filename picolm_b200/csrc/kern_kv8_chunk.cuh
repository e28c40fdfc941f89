// kern_kv8_chunk.cuh -- causal attention of several tokens a slot over the
// 8-bit paged cache, on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// Bound by the softmax (its exponentials and the work around them) and, for
// FP32 activations, by the tensor pipe, which then runs every product twice
// (high part and residual).
//
// Work.  A query item is up to two 128-row tiles ("slots" A and B) of one
// entry and KV head: row r of a slot is token r / G, query head r % G of the
// G heads that share the KV head, so a few tokens already fill a tile and
// both slots read the same K/V tiles.  The (item, K/V tile) pairs of all
// entries, in order, form one list, and every block (one per SM) takes an
// equal contiguous slice of it: long prompts balance by themselves, and few
// tokens over a long context are split along it.  The part of an item in a
// slice is a segment; an item over several blocks leaves one partial (m, l,
// o) a block in the workspace, and the block that leaves the last one merges
// them in the order of the blocks.  Every role of the block derives the same
// sequence of segments from the entries' prefix sums.
//
// Roles (512 threads = four warpgroups):
//   warps 0-3, 4-7   softmax of slots A, B; thread r owns query row r =
//                    TMEM lane r: it rotates, scales and splits its row of q
//                    into shared memory, and per tile turns S into weights
//   warps 8-11       producers: fetch the codes of a K/V tile from the pages
//                    (one tile ahead, in registers), write them as FP16 --
//                    every code is exact -- into a ring of swizzled tiles
//   warps 12, 13     MMA issuers of slots A, B (12 allocates TMEM)
//   warps 14, 15     idle (they complete the warpgroup)
// Per tile j the issuer of slot x issues S_x(j) = Q_x K_j^T and then
// O_x += P_x(j-1) V, so a slot's softmax overlaps its own next scores and
// the other slot's products.
//
// Scales and ranges.  K's scale multiplies 16 columns of S before the row
// maximum; V's goes into the weight, relative to a reference that is raised
// (with O rescaled) when a scale outgrows it fourfold, as the running
// maximum is when a score outgrows it by 2^8, so weights stay below 2^14.
// q is scaled by a power of two a row.  FP32 activations (PARTS 2): q and
// the weights are FP16 high part + residual.  Sixteen-bit ones (PARTS 1):
// q and the weights are rounded to FP16 once, 2^-12 relative, half or less of
// what rounding the output to its type costs.
#pragma once
#include <cstdint>
#include <cuda.h>

#include "kern_kv8_attn.cuh"

namespace pl {

constexpr int kChRows = 128;       // query rows of a slot
constexpr int kChThreads = 512;
constexpr int kChLaunchRegs = 128;
constexpr int kChSoftmaxRegs = 192;
constexpr int kChProducerRegs = 80;
constexpr int kChOtherRegs = 48;
static_assert(256 * kChSoftmaxRegs + 128 * kChProducerRegs + 128 * kChOtherRegs <=
                  kChThreads * kChLaunchRegs,
              "register split exceeds the launch allocation");
constexpr int kChMinTiles = 4;         // K/V tiles of a block's slice, at least
constexpr float kChBase = 16.f;        // weight of a row's maximum under the largest scale
constexpr float kChRescaleLog2 = 8.f;  // raise the running maximum only past 2^8
constexpr float kChRefGrowth = 4.f;    // raise the scale reference only past 4x

template <int HD, int PARTS>
struct ChShape {
  static constexpr int kBN = HD == 64 && PARTS == 1 ? 128 : 64;  // rows of a K/V tile
  static constexpr int kHalves = HD / 64;          // 64-element (128-byte) halves of a row
  static constexpr int kQHalf = kChRows * 128;
  static constexpr int kQBytes = kQHalf * kHalves;
  static constexpr int kKVHalf = kBN * 128;
  static constexpr int kKVBytes = kKVHalf * kHalves;
  static constexpr int kStages = HD == 128 && PARTS == 2 ? 2 : 3;
  static constexpr int kPages = kBN / kPage;       // pages of a tile
  static constexpr int kBlocks = kBN / kBlock;     // scales of a tile, of K and of V
  // TMEM columns: S_A, S_B (kBN FP32 each), O_A, O_B (HD), P_A, P_B (kBN/2 a part)
  static constexpr int kPCols = kBN / 2 * PARTS;
  static __device__ __forceinline__ uint32_t col_s(int x) { return x * kBN; }
  static __device__ __forceinline__ uint32_t col_o(int x) { return 2 * kBN + x * HD; }
  static __device__ __forceinline__ uint32_t col_p(int x) {
    return 2 * kBN + 2 * HD + x * kPCols;
  }
  static_assert(2 * kBN + 2 * HD + 2 * kPCols <= 512, "TMEM columns");
  static constexpr int kPartFloats = 2 * kChRows * (HD + 2);  // a partial: [slot][o.., m, l][row]
};

template <int HD, int PARTS>
struct ChSmem {
  using Sh = ChShape<HD, PARTS>;
  // 1024-byte aligned tiles (128-byte swizzle)
  uint8_t q[2][PARTS][Sh::kQBytes];
  uint8_t k[Sh::kStages][Sh::kKVBytes];
  uint8_t v[Sh::kStages][Sh::kKVBytes];
  float scale[Sh::kStages][2][Sh::kBlocks];
  double half_turns[HD / 2];
  long long prefix[kPlanSeqs + 1];
  int slot[kPlanSeqs], len[kPlanSeqs], tok0[kPlanSeqs], n_tok[kPlanSeqs];
  uint64_t q_full[2], kv_full[Sh::kStages], kv_empty[Sh::kStages];
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2][2], mma_done[2];
  long long warp_sum[kChThreads / 32];
  uint32_t tmem_base;
  int merge;
};

struct Kv8ChunkArgs {
  Kv8AttnArgs a;
  float* part;   // [2 * blocks][kPartFloats]
  int* arrived;  // [blocks], zero at rest: by the block where an item starts
};

// K/V tiles of query item t of an entry (at least one, which may be all
// masked, so that rows with nothing to attend are written).
struct ChEntry {
  int len, n_tok, per_item;  // rows; query tokens; tokens of an item (both slots)
};
template <int BN>
__device__ __forceinline__ int ch_tiles(const ChEntry& e, int t) {
  const int last = e.len - e.n_tok + min(e.n_tok, (t + 1) * e.per_item) - 1;
  return last < 0 ? 1 : last / BN + 1;
}

// A row of q, rotated by its position (all of it in registers: indexes are
// compile-time).
template <typename T, int HD>
__device__ __forceinline__ void load_q_row(const T* q, int pos, const pl_rope& rope,
                                           const double* half_turns, float (&y)[HD]) {
#pragma unroll
  for (int d = 0; d < HD; d += 8) load8(q + d, *reinterpret_cast<float(*)[8]>(y + d));
  const int half = rope.dim >> 1;
  if (rope.type == PL_ROPE_LLAMA) {
#pragma unroll
    for (int i = 0; i < HD / 2; ++i)
      if (i < half) {
        const float2 f = rope_cs_fast(half_turns[i], rope.gain, pos);
        const float u = y[2 * i], v = y[2 * i + 1];
        y[2 * i] = u * f.x - v * f.y;
        y[2 * i + 1] = u * f.y + v * f.x;
      }
  } else if (rope.dim == HD) {
#pragma unroll
    for (int i = 0; i < HD / 2; ++i) {
      const float2 f = rope_cs_fast(half_turns[i], rope.gain, pos);
      const float u = y[i], v = y[i + HD / 2];
      y[i] = u * f.x - v * f.y;
      y[i + HD / 2] = u * f.y + v * f.x;
    }
  } else {  // part of the head: the partner's place is not known here
#pragma unroll
    for (int d = 0; d < HD; ++d)
      if (d < rope.dim) {
        const float2 f = rope_cs_fast(half_turns[d < half ? d : d - half], rope.gain, pos);
        const float o = to_f32(q[d < half ? d + half : d - half]);
        y[d] = d < half ? y[d] * f.x - o * f.y : o * f.y + y[d] * f.x;
      }
  }
}

// The sequence of segments of a block's slice [x, x1).
template <int BN>
struct ChWalk {
  long long x, x1;      // next tile of the list, end of the slice
  int i, h, t, j;       // entry, KV head, item, next tile of the item
  int n_items;          // items of the entry
  ChEntry e;
  // the current segment
  int si, sh, stt, j0, j1, tiles;
  long long item_first;  // list position of the item's first tile
};

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kChThreads, 1) kv8_chunk_kernel(
    const __grid_constant__ Kv8ChunkArgs ca) {
  constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
  using Sh = ChShape<HD, PARTS>;
  constexpr int BN = Sh::kBN, NS = Sh::kStages;
  extern __shared__ uint8_t smem_raw[];
  ChSmem<HD, PARTS>& sm = *reinterpret_cast<ChSmem<HD, PARTS>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const Kv8AttnArgs& a = ca.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = a.g.n_kv_heads, G = a.group;
  const int slot_tok = kChRows / G, per_item = 2 * slot_tok;

  if (tid < HD / 2) sm.half_turns[tid] = a.rope.half_turns[tid];
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&sm.kv_full[s], 4);   // one arrival per producer warp
      mbar_init(&sm.kv_empty[s], 2);  // one per issuer
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
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- tiles of every entry, scanned
  for (int i = warp; i < a.n; i += kChThreads / 32) {
    Kv8Entry en;
    const bool ok = kv8_entry(a.g, i, a.total, a.max_tok, a.seqs, a.start, en);
    if (!ok && blockIdx.x == 0 && lane == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    const ChEntry e{ok ? en.len : 0, ok ? en.n_tok : 0, per_item};
    long long units = 0;
    for (int t = lane; t * per_item < e.n_tok; t += 32) units += ch_tiles<BN>(e, t);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) units += __shfl_xor_sync(0xffffffffu, units, d);
    if (lane == 0) {
      sm.slot[i] = en.slot;
      sm.len[i] = e.len;
      sm.tok0[i] = en.tok0;
      sm.n_tok[i] = e.n_tok;
      sm.prefix[i] = units * heads;
    }
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
    long long base = 0, total = 0;
    for (int w = 0; w < kChThreads / 32; ++w) {
      base += w < warp ? sm.warp_sum[w] : 0;
      total += sm.warp_sum[w];
    }
    long long run = base + x - mine;
    for (int i = i0; i < min(a.n, i0 + per); ++i) {
      const long long u = sm.prefix[i];
      sm.prefix[i] = run;
      run += u;
    }
    if (tid == 0) sm.prefix[a.n] = total;
    __syncthreads();
  }
  const uint32_t tmem = sm.tmem_base;
  const long long total = sm.prefix[a.n];
  // a few tiles a block at least: a split costs its merge
  const long long most = (total + kChMinTiles - 1) / kChMinTiles;
  const long long blocks = most < gridDim.x ? most : gridDim.x;
  const int blk = blockIdx.x;
  auto begin = [&](long long b) { return b * total / blocks; };
  auto block_of = [&](long long x) { return static_cast<int>(((x + 1) * blocks - 1) / total); };
  const bool works = blk < blocks;
  const long long b0 = works ? begin(blk) : 0, b1 = works ? begin(blk + 1) : 0;

  ChWalk<BN> wk;
  wk.x = b0;
  wk.x1 = b1;
  if (works) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sm.prefix[mid + 1] > b0) hi = mid; else lo = mid + 1;
    }
    wk.i = lo;
    wk.e = ChEntry{sm.len[lo], sm.n_tok[lo], per_item};
    wk.n_items = (wk.e.n_tok + per_item - 1) / per_item;
    const long long per_head = (sm.prefix[lo + 1] - sm.prefix[lo]) / heads;
    long long rem = b0 - sm.prefix[lo];
    wk.h = static_cast<int>(rem / per_head);
    rem -= wk.h * per_head;
    wk.t = 0;
    while (rem >= ch_tiles<BN>(wk.e, wk.t)) rem -= ch_tiles<BN>(wk.e, wk.t++);
    wk.j = static_cast<int>(rem);
  }
  // The next segment of the slice; false at its end.
  auto next = [&]() -> bool {
    if (wk.x >= wk.x1) return false;
    wk.tiles = ch_tiles<BN>(wk.e, wk.t);
    wk.si = wk.i, wk.sh = wk.h, wk.stt = wk.t, wk.j0 = wk.j;
    wk.item_first = wk.x - wk.j;
    const long long left = wk.x1 - wk.x;
    wk.j1 = left < wk.tiles - wk.j ? wk.j + static_cast<int>(left) : wk.tiles;
    wk.x += wk.j1 - wk.j0;
    wk.j = 0;
    if (++wk.t == wk.n_items) {
      wk.t = 0;
      if (++wk.h == heads) {
        wk.h = 0;
        do ++wk.i; while (wk.i < a.n && sm.n_tok[wk.i] == 0);
        if (wk.i < a.n) {
          wk.e = ChEntry{sm.len[wk.i], sm.n_tok[wk.i], per_item};
          wk.n_items = (wk.e.n_tok + per_item - 1) / per_item;
        }
      }
    }
    return true;
  };

  if (warp >= 12) {
    regs_dec<kChOtherRegs>();
    if (warp < 14 && lane == 0) {
      // ------------------------------------------------- MMA issuer of slot x
      const int x = warp - 12;
      const uint32_t idesc_qk = idesc_f16_f32(128, BN, 0);
      const uint32_t idesc_pv = idesc_f16_f32(128, 64, 1);
      const uint32_t q_addr = smem_u32(sm.q[x][0]);
      int J = 0, A = 0, k = 0;  // tiles of the block, tiles and segments of this slot
      bool ok = true;
      auto issue_pv = [&](int g, int n, bool first) -> bool {  // block's tile g, slot's tile n
        const int s = g % NS, pb = n & 1;
        if (!mbar_wait_bounded(&sm.p_full[x][pb], (n >> 1) & 1)) return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sm.v[s]);
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
                        (first && part == 0 && kk == 0) ? 0u : 1u);
            }
        tc_commit(&sm.pv_done[x][pb]);
        tc_commit(&sm.kv_empty[s]);
        return true;
      };
      while (ok && next()) {
        const int nt = wk.j1 - wk.j0;
        if (wk.stt * per_item + x * slot_tok >= sm.n_tok[wk.si]) {
          // this slot has no token in the item: it only frees the stages
          for (int j = 0; j < nt && ok; ++j) {
            const int g = J + j;
            if (!mbar_wait_bounded(&sm.kv_full[g % NS], (g / NS) & 1)) ok = false;
            else mbar_arrive(&sm.kv_empty[g % NS]);
          }
          J += nt;
          continue;
        }
        if (!mbar_wait_bounded(&sm.q_full[x], k & 1)) { ok = false; break; }
        for (int j = 0; j < nt && ok; ++j) {
          const int g = J + j, n = A + j, s = g % NS;
          if (!mbar_wait_bounded(&sm.kv_full[s], (g / NS) & 1)) { ok = false; break; }
          if (n >= 1 && !mbar_wait_bounded(&sm.s_free[x], (n - 1) & 1)) { ok = false; break; }
          tc_fence_after();
          const uint32_t k_addr = smem_u32(sm.k[s]);
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
          if (j >= 1 && !issue_pv(g - 1, n - 1, j == 1)) ok = false;
        }
        if (ok && !issue_pv(J + nt - 1, A + nt - 1, nt == 1)) ok = false;
        J += nt;
        A += nt;
        ++k;
      }
      if (!ok) atomicOr(&a.g.head->err, ERR_TIMEOUT_MMA);
      // all issued MMAs must finish before TMEM is freed
      tc_commit(&sm.mma_done[x]);
      mbar_wait_bounded(&sm.mma_done[x], 0);
    }
  } else if (warp >= 8) {
    regs_dec<kChProducerRegs>();
    // ------------------------------------------------------------ producers
    const int pt = tid - 256;
    constexpr int kChunks = BN * HD / 16 / 128;  // 16-byte chunks a thread, of K and of V
    constexpr int kPerRow = HD / 16;
    const int ch = pt % kPerRow;
    uint4 ck[kChunks], cv[kChunks];
    float sc = 0.f;
    int J = 0;
    bool ok = true;
    // The codes and scales of tile j of the current segment's item.
    auto fetch = [&](int j) {
      const int len = sm.len[wk.si];
      const int* row_table = a.g.table + static_cast<long long>(sm.slot[wk.si]) * a.g.max_pages;
      int pages[Sh::kPages];
#pragma unroll
      for (int p = 0; p < Sh::kPages; ++p) {
        const int at = j * Sh::kPages + p;
        pages[p] = at * kPage < len ? row_table[at] : 0;
        if (pages[p] < 0 || pages[p] >= a.g.n_pages) {
          if (pt == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
          pages[p] = 0;
        }
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int row = (c * 128 + pt) / kPerRow;  // of the tile
        const int page = Sh::kPages == 1 || c < kChunks / 2 ? pages[0] : pages[Sh::kPages - 1];
        const uint8_t* src =
            a.g.codes + (a.g.slab(page, wk.sh, 0) * kPage + row % kPage) * HD + ch * 16;
        ck[c] = cv[c] = make_uint4(0, 0, 0, 0);
        if (j * BN + row < len) {
          ck[c] = __ldg(reinterpret_cast<const uint4*>(src));
          cv[c] = __ldg(reinterpret_cast<const uint4*>(src + kPage * HD));
        }
      }
      if (pt < 2 * Sh::kBlocks) {
        const int kv = pt / Sh::kBlocks, b = pt % Sh::kBlocks;
        const int page = pages[Sh::kPages == 1 ? 0 : b / kBlocksPerPage];
        sc = 0.f;
        if (j * BN + b * kBlock < len)
          sc = __ldg(a.g.scales + a.g.slab(page, wk.sh, kv) * kBlocksPerPage + b % kBlocksPerPage);
      }
    };
    auto put = [&](uint8_t* tile, const uint4& w, int row) {
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      uint32_t o[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        o[2 * q] = codes_half2<FMT, 0x10>(in[q]);
        o[2 * q + 1] = codes_half2<FMT, 0x32>(in[q]);
      }
      // elements 16 ch .. of the row: chunks 2ch, 2ch + 1 of its 64-element halves
      const uint32_t base = smem_u32(tile) + (ch >> 2) * Sh::kKVHalf + row * 128;
      const int c0 = 2 * (ch & 3);
#pragma unroll
      for (int q = 0; q < 2; ++q)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                         base + (((c0 + q) ^ (row & 7)) << 4)),
                     "r"(o[4 * q]), "r"(o[4 * q + 1]), "r"(o[4 * q + 2]), "r"(o[4 * q + 3])
                     : "memory");
    };
    bool have = next();
    int j = have ? wk.j0 : 0;
    if (have) fetch(j);
    while (have && ok) {
      const int s = J % NS;
      if (J >= NS && !mbar_wait_bounded(&sm.kv_empty[s], ((J / NS) - 1) & 1)) {
        if (lane == 0) atomicOr(&a.g.head->err, ERR_TIMEOUT_EMPTY);
        ok = false;
        break;
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int row = (c * 128 + pt) / kPerRow;
        put(sm.k[s], ck[c], row);
        put(sm.v[s], cv[c], row);
      }
      if (pt < 2 * Sh::kBlocks) sm.scale[s][pt / Sh::kBlocks][pt % Sh::kBlocks] = sc;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.kv_full[s]);
      ++J;
      if (++j == wk.j1) {
        have = next();
        j = have ? wk.j0 : 0;
      }
      if (have) fetch(j);
    }
  } else {
    regs_inc<kChSoftmaxRegs>();
    // -------------------------------------------------------------- softmax
    const int x = warp >> 2;        // slot
    const int r = tid & 127;        // query row of the slot, TMEM lane
    const int row_tok = r / G, row_head = r - row_tok * G;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int J = 0, A = 0;
    // a wait that gave up ends this warp's work, but not its part in the
    // barriers of the segments
    bool ok = true;
    while (next()) {
      const int i = wk.si, nt = wk.j1 - wk.j0;
      const int tok_x = wk.stt * per_item + x * slot_tok;  // the slot's first token
      const bool active = ok && tok_x < sm.n_tok[i];
      const bool whole = nt == wk.tiles;
      const int tok = tok_x + row_tok;
      const bool real = row_tok < slot_tok && tok < sm.n_tok[i];
      const int p_min = sm.len[i] - sm.n_tok[i] + tok_x;   // position of the slot's first token
      const int pos = real ? p_min + row_tok : -1;
      float m_used = -INFINITY, l_run = 0.f, ref = kMinRef, q_scale = 0.f;
      const long long out_row = static_cast<long long>(sm.tok0[i]) + tok;
      const int head_el = (wk.sh * G + row_head) * HD;
      if (active) {
        // ---- this thread's row of q: rotated, scaled, split, into the tile
        float y[HD];
        if (real) {
          const T* q = static_cast<const T*>(a.q) + out_row * a.q_stride + head_el;
          load_q_row<T, HD>(q, max(pos, 0), a.rope, sm.half_turns, y);
        } else {
#pragma unroll
          for (int d = 0; d < HD; ++d) y[d] = 0.f;
        }
        float top = 0.f;
#pragma unroll
        for (int d = 0; d < HD; ++d) top = fmaxf(top, fabsf(y[d]));
        const uint32_t ex = __float_as_uint(top) >> 23;
        const bool norm = ex > 1 && ex < 253;
        const float down = norm ? __uint_as_float((254u - ex) << 23) : 1.f;
        q_scale = (norm ? __uint_as_float(ex << 23) : 1.f) * a.score_scale;
#pragma unroll
        for (int c8 = 0; c8 < HD / 8; ++c8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = y[8 * c8 + 2 * e] * down, v = y[8 * c8 + 2 * e + 1] * down;
            if constexpr (PARTS == 2) split_hi_lo(u, v, hi[e], lo[e]);
            else hi[e] = pack_half2(u, v);
          }
          const uint32_t off =
              (c8 >> 3) * Sh::kQHalf + r * 128 + (((c8 & 7) ^ (r & 7)) << 4);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(sm.q[x][0]) + off),
                       "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3])
                       : "memory");
          if constexpr (PARTS == 2)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                             smem_u32(sm.q[x][PARTS - 1]) + off),
                         "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3])
                         : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[x]);
        for (int j = 0; j < nt; ++j) {
          const int g = J + j, n = A + j, s = g % NS;
          // (the tile's scales are the producers' writes)
          if (!mbar_wait_bounded(&sm.kv_full[s], (g / NS) & 1) ||
              !mbar_wait_bounded(&sm.s_full[x], n & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t sv[BN];
#pragma unroll
          for (int c4 = 0; c4 < BN / 32; ++c4)
            tc_ld_32x32b_x32(lane_base + Sh::col_s(x) + 32 * c4,
                             *reinterpret_cast<uint32_t(*)[32]>(sv + 32 * c4));
          tc_wait_ld();
#pragma unroll
          for (int d = 0; d < BN; ++d) asm volatile("" : "+r"(sv[d]));
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.s_free[x]);
          const int t0 = (wk.j0 + j) * BN;
          const bool need_mask = t0 + BN - 1 > p_min;
          const int lim = pos - t0;  // columns c <= lim are visible
          const float* sk = sm.scale[s][0];
          const float* svs = sm.scale[s][1];
#pragma unroll
          for (int b = 0; b < Sh::kBlocks; ++b) {
            const float2 by = make_float2(sk[b], sk[b]);
#pragma unroll
            for (int c = 16 * b; c < 16 * b + 16; c += 2) {
              const float2 v =
                  mul2(make_float2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), by);
              sv[c] = __float_as_uint(v.x);
              sv[c + 1] = __float_as_uint(v.y);
            }
          }
          if (need_mask) {
#pragma unroll
            for (int c = 0; c < BN; ++c)
              if (c > lim) sv[c] = __float_as_uint(-INFINITY);
          }
          float mp[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) mp[u] = __uint_as_float(sv[u]);
#pragma unroll
          for (int c = 8; c < BN; c += 8)
#pragma unroll
            for (int u = 0; u < 8; ++u) mp[u] = fmaxf(mp[u], __uint_as_float(sv[c + u]));
          const float m_tile = max3(max3(mp[0], mp[1], mp[2]), max3(mp[3], mp[4], mp[5]),
                                    fmaxf(mp[6], mp[7])) * q_scale;
          float top_v = svs[0];
#pragma unroll
          for (int b = 1; b < Sh::kBlocks; ++b) top_v = fmaxf(top_v, svs[b]);
          const bool rescale = __any_sync(0xffffffffu, m_tile > m_used + kChRescaleLog2) ||
                               top_v > kChRefGrowth * ref;
          float keep = 1.f;
          if (rescale) {
            const float m_new = fmaxf(m_used, m_tile);
            const float alpha = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
            const float ref_new = fmaxf(ref, top_v);
            l_run *= alpha;
            keep = alpha * (ref / ref_new);
            m_used = m_new;
            ref = ref_new;
          }
          const float lift = kChBase / ref;
          const float m_safe = m_used == -INFINITY ? 0.f : m_used;
          const float2 sc2 = make_float2(q_scale, q_scale), nm2 = make_float2(-m_safe, -m_safe);
          float2 rs2[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) rs2[e] = make_float2(0.f, 0.f);
#pragma unroll
          for (int q = 0; q < BN / 32; ++q) {  // 32 columns: 16 TMEM columns a part
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int c = 32 * q + 2 * e;
              const float2 arg =
                  fma2(make_float2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), sc2, nm2);
              const float2 p = make_float2(ex2(arg.x), ex2(arg.y));
              rs2[e & 3] = add2(rs2[e & 3], p);
              const float by = svs[c / kBlock] * lift;
              float2 w = mul2(p, make_float2(by, by));
              if (need_mask) {  // a masked column's scale may be NaN
                w.x = c > lim ? 0.f : w.x;
                w.y = c + 1 > lim ? 0.f : w.y;
              }
              if constexpr (PARTS == 2) split_hi_lo(w.x, w.y, hi[e], lo[e]);
              else hi[e] = pack_half2(w.x, w.y);
            }
            if (q == 0) {
              // P(n) overwrites P(n-1) and O is rescaled: both need PV(n-1) done
              if (n >= 1 && !mbar_wait_bounded(&sm.pv_done[x][(n - 1) & 1], ((n - 1) >> 1) & 1)) {
                ok = false;
                break;
              }
              tc_fence_after();
              if (rescale && j >= 1) {
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
            tc_st_32x32b_x16(lane_base + Sh::col_p(x) + 16 * q, hi);
            if constexpr (PARTS == 2)
              tc_st_32x32b_x16(lane_base + Sh::col_p(x) + BN / 2 + 16 * q, lo);
          }
          if (!ok) break;
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[x][n & 1]);
          const float2 ra = add2(rs2[0], rs2[1]), rb = add2(rs2[2], rs2[3]);
          l_run += (ra.x + ra.y) + (rb.x + rb.y);
        }
        // ---- the segment's O
        const int last = A + nt - 1;
        ok = ok && mbar_wait_bounded(&sm.pv_done[x][last & 1], (last >> 1) & 1);
        tc_fence_after();
        A += nt;
      }
      float* part = nullptr;
      const int kind = wk.j0 > 0 ? 0 : 1;
      if (!whole)
        part = ca.part + static_cast<long long>(2 * blk + kind) * Sh::kPartFloats +
               static_cast<long long>(x) * kChRows * (HD + 2) + r;
      if (active && ok) {
        const float back = ref * (1.f / kChBase);
        const float by = whole ? (l_run == 0.f ? 0.f : back / l_run) : back;
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += 32) {
          uint32_t ov[32];
          tc_ld_32x32b_x32(lane_base + Sh::col_o(x) + d0, ov);
          tc_wait_ld();
#pragma unroll
          for (int d = 0; d < 32; ++d) asm volatile("" : "+r"(ov[d]));
          if (whole) {
            if (real) {
              T* dst = static_cast<T*>(a.out) + out_row * a.out_stride + head_el + d0;
#pragma unroll
              for (int d = 0; d < 32; d += 8) {
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = __uint_as_float(ov[d + e]) * by;
                store8(dst + d, z);
              }
            }
          } else {
#pragma unroll
            for (int d = 0; d < 32; ++d)
              part[(d0 + d) * kChRows] = __uint_as_float(ov[d]) * by;
          }
        }
        tc_fence_before();
        if (!whole) {
          part[HD * kChRows] = m_used;
          part[(HD + 1) * kChRows] = l_run;
        }
      }
      if (!whole) {
        // ---- leave the partial; the last block of the item merges them
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int f0 = block_of(wk.item_first);
        const int parts = block_of(wk.item_first + wk.tiles - 1) - f0 + 1;
        if (tid == 0) {
          const bool done = atomicAdd(&ca.arrived[f0], 1) == parts - 1;
          if (done) ca.arrived[f0] = 0;
          sm.merge = done;
          __threadfence();
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (sm.merge && active && real) {
          const long long stride = static_cast<long long>(2) * Sh::kPartFloats;
          // the first block's partial is of kind 1, the others' of kind 0
          const float* p0 = ca.part + static_cast<long long>(2 * f0) * Sh::kPartFloats +
                            static_cast<long long>(x) * kChRows * (HD + 2) + r;
          auto at = [&](int p) { return p0 + p * stride + (p == 0 ? Sh::kPartFloats : 0); };
          float M = -INFINITY, L = 0.f;
          for (int p = 0; p < parts; ++p) M = fmaxf(M, __ldcg(at(p) + HD * kChRows));
          const float Ms = M == -INFINITY ? 0.f : M;
          for (int p = 0; p < parts; ++p)
            L += ex2(__ldcg(at(p) + HD * kChRows) - Ms) * __ldcg(at(p) + (HD + 1) * kChRows);
          const float inv = L == 0.f ? 0.f : 1.f / L;
          T* dst = static_cast<T*>(a.out) + out_row * a.out_stride + head_el;
#pragma unroll 1
          for (int d0 = 0; d0 < HD; d0 += 32) {
            float z[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) z[d] = 0.f;
            for (int p = 0; p < parts; ++p) {
              const float w = ex2(__ldcg(at(p) + HD * kChRows) - Ms) * inv;
#pragma unroll
              for (int d = 0; d < 32; ++d) z[d] += w * __ldcg(at(p) + (d0 + d) * kChRows);
            }
#pragma unroll
            for (int d = 0; d < 32; d += 8)
              store8(dst + d0 + d, *reinterpret_cast<float(*)[8]>(z + d));
          }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      J += nt;
    }
    if (!ok) atomicOr(&a.g.head->err, ERR_TIMEOUT_MMA);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace pl
