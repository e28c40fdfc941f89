// kern_kv8.cuh -- the 8-bit paged KV cache: appending rows, reading them
// back, and the books and copies of its pages.
//
// Layout.  codes [page][layer][kv head][K, V][64 rows][head_dim] bytes and
// scales [page][layer][kv head][K, V][4] FP32, one scale for each block of
// 16 rows: a value is code * scale.  A page is contiguous over its layers,
// so copying one is one long run; one head's K and V rows of a page are
// contiguous, so attention fetches a page and head with a few bulk copies.
// Blocks of 16 rows are the K extent of one mma.sync / tcgen05.mma step, so
// a scale is constant within a step and multiplies the score (K) or the
// softmax weight (V) instead of every element.
#pragma once
#include <cstdint>
#include <cuda_fp8.h>

#include "kern_rope.cuh"
#include "sm100.cuh"

namespace pl {

constexpr int kPage = PL_KV8_PAGE;    // rows per page
constexpr int kBlock = PL_KV8_BLOCK;  // rows per scale
constexpr int kBlocksPerPage = kPage / kBlock;

// Additional bit of the error word of a cache (see sm100.cuh).
enum : uint32_t { ERR_NO_PAGES = 16u };

// Header of the caller's workspace.
struct Kv8Head {
  uint32_t err;
  uint32_t n_copies;  // pages that the plan kernel wants copied
  uint32_t pad[62];
};

// What every kernel of the cache needs of pl_kv8.
struct Kv8Geo {
  uint8_t* codes;
  float* scales;
  int* table;
  int* lens;
  int* refs;
  Kv8Head* head;
  int n_layers, n_kv_heads, n_pages, n_seqs, max_pages, layer;

  // (page, layer, head, K or V) as one index: codes at 64 * head_dim * slab
  // bytes, scales at 4 * slab
  __device__ __forceinline__ long long slab(int page, int h, int kv) const {
    return ((static_cast<long long>(page) * n_layers + layer) * n_kv_heads + h) * 2 + kv;
  }
};

// ---------------------------------------------------------------- codes
// Largest code and rounding of the two formats.
template <int FMT>
__device__ __forceinline__ float code_top() {
  return FMT == PL_KV8_INT8 ? 127.f : 448.f;
}

// Eight values, already divided by their scale, as codes: rounded to
// nearest (halves to even), saturated.
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&x)[8]) {
  uint32_t w[2];
  if constexpr (FMT == PL_KV8_INT8) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t b = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = __float2int_rn(fminf(fmaxf(x[4 * j + e], -127.f), 127.f));
        b |= (static_cast<uint32_t>(v) & 0xffu) << (8 * e);
      }
      w[j] = b;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j], x[4 * j + 1]),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j + 2], x[4 * j + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
      w[j] = lo | (hi << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

template <int FMT>
__device__ __forceinline__ void decode8(uint2 c, float (&x)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (FMT == PL_KV8_INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[4 * j + e] = static_cast<float>(static_cast<int>(w[j] << (24 - 8 * e)) >> 24);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
            static_cast<__nv_fp8x2_storage_t>(w[j] >> (16 * e)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        x[4 * j + 2 * e] = f.x;
        x[4 * j + 2 * e + 1] = f.y;
      }
    }
  }
}

// ---------------------------------------------------------------- append
struct Kv8AppendArgs {
  Kv8Geo g;
  pl_rope rope;
  int n, total, max_tok;
  const int* seqs;
  const int* start;  // [n + 1] first token of each sequence; nullptr: one token each
  const void *k, *v;
  long long k_stride, v_stride;
};

// Slot, row range and tokens of entry i of a call; false (with the error
// recorded by one thread) when they are out of range.
struct Kv8Entry {
  int slot, len, tok0, n_tok;
};
__device__ __forceinline__ bool kv8_entry(const Kv8Geo& g, int i, int total, int max_tok,
                                          const int* seqs, const int* start, Kv8Entry& e) {
  e.slot = seqs[i];
  e.tok0 = start ? start[i] : i;
  e.n_tok = start ? start[i + 1] - e.tok0 : 1;
  if (e.slot < 0 || e.slot >= g.n_seqs || e.tok0 < 0 || e.n_tok < 0 || e.n_tok > max_tok ||
      e.tok0 > total - e.n_tok)
    return false;
  e.len = g.lens[e.slot];
  return e.len >= 0 && e.len <= g.max_pages * kPage;
}

constexpr int kAppendThreads = 256;

// Elements [e, e + 8) of a head row as they are, and the run that rotates
// with them (Qwen).
template <typename T>
__device__ __forceinline__ void load_pair8(const T* x, int e, const pl_rope& r, bool rotated,
                                           Raw8<T>& y, Raw8<T>& z) {
  y = raw8(x + e);
  if (!rotated || r.type == PL_ROPE_LLAMA || e >= r.dim) return;
  const int half = r.dim >> 1;
  if (half % 8 == 0) {
    z = raw8(x + (e < half ? e + half : e - half));
  } else {
    T* p = reinterpret_cast<T*>(&z);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = e + j;
      p[j] = x[d < half ? d + half : d < r.dim ? d - half : d];
    }
  }
}
// y rotated by cs[place of the pair], with the roundings of rope().
template <int HD>
__device__ __forceinline__ void rotate_pair8(int e, const pl_rope& r, const float2* cs,
                                             float (&y)[8], const float (&z)[8]) {
  if (e >= r.dim) return;
  const int half = r.dim >> 1;
  if (r.type == PL_ROPE_LLAMA) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e + 2 * j < r.dim)
        rope_one(y[2 * j], y[2 * j + 1], cs[pair_place<true>((e >> 1) + j, HD / 2)]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = e + j;
      if (d >= r.dim) break;
      const float2 f = cs[pair_place<false>(d < half ? d : d - half, HD / 2)];
      y[j] = d < half ? __fsub_rn(__fmul_rn(y[j], f.x), __fmul_rn(z[j], f.y))
                      : __fadd_rn(__fmul_rn(z[j], f.y), __fmul_rn(y[j], f.x));
    }
  }
}

// x / by, correctly rounded, from the rounded reciprocal inv of by
// (Markstein, 1990: one correction by the exact remainder gives the rounded
// quotient), where nothing comes near the ends of the range.  0 for -0.
__device__ __forceinline__ float quotient(float x, float by, float inv) {
  const float q = __fmul_rn(x, inv);
  return fmaf(fmaf(-q, by, x), inv, q);
}

// Block (x, y) of the grid: the x-th block of 16 rows that entry y touches,
// all heads, K and V.  A warp takes one (head, K or V): its 16 rows live in
// registers from the absolute maximum to the codes, so every input is read
// once.  The block's scale is its largest absolute value over the largest
// code; rows that the block held before are kept, rescaled when the new
// rows raise the scale (code' = round(code * old / new)).  A row with a
// NaN or infinity makes the scale NaN: the whole block then reads as NaN
// rather than as finite numbers that were never written.  Its new codes are 0:
// e4m3 has a code for NaN, and attention multiplies the codes of rows that a
// mask hides by a weight of 0, which a NaN would survive.
//
// Cosines are FP64 and rounded once; a block of rows takes a sincospi or two a
// pair (its first row's and one row's step) and turns from row to row by FP64
// products.  A call of one token takes a sincospi of the row itself, as the
// decode step does; the two are apart by up to (position + 32) 2^-52 (for
// frequencies up to 1), so how rows were appended can move a cosine by one
// rounding to FP32 where it lies that near to a border.  And rows that came one
// by one have been rounded again each time the scale of their block grew.
//
// Should be bound by HBM, is bound by instructions and the latency of few
// warps (51% of the issue slots, at 18 warps an SM): 8
// prompts of up to 4096 BF16 rows of 8 heads of 128 to e4m3 (157 MB) take 94
// us, 1.7 TB/s.  On the way, with reading them back (33 us): a sincospi a row
// and pair and a division an element 330 us; without them 238; rows fetched
// as raw 16-byte runs ahead of their use 174; tables free of bank conflicts
// 143; 32 values a lane instead of 64, and so three blocks an SM instead of
// two, 125.
// 64 rows of a decode step: 6.7 us, a chain of dependent loads (books, rows,
// scale).
template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kAppendThreads, 3) kv8_append_kernel(
    const __grid_constant__ Kv8AppendArgs a) {
  __shared__ float2 s_cs[kBlock][HD / 2];
  __shared__ double s_turns[HD / 2];
  __shared__ uint32_t s_top[2][kAppendThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < HD / 2) s_turns[threadIdx.x] = a.rope.half_turns[threadIdx.x];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Kv8Entry e;
  if (!kv8_entry(a.g, blockIdx.y, a.total, a.max_tok, a.seqs, a.start, e) || e.len < e.n_tok) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    return;
  }
  const int row0 = e.len - e.n_tok;                       // first new row
  const int blk = row0 / kBlock + blockIdx.x;             // block of the sequence
  if (e.n_tok == 0 || blk * kBlock >= e.len) return;
  const int page = a.g.table[static_cast<long long>(e.slot) * a.g.max_pages + blk / kBlocksPerPage];
  if (page < 0 || page >= a.g.n_pages) {
    if (threadIdx.x == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    return;
  }
  const int lo = max(row0 - blk * kBlock, 0), hi = min(e.len - blk * kBlock, kBlock);  // new rows
  const int pairs = a.rope.dim >> 1;
  __syncthreads();
  {
    // thread (pair, group): rows lo + group * per .. of the pair
    constexpr int kGroups = kAppendThreads / (HD / 2);
    const int i = threadIdx.x % (HD / 2), group = threadIdx.x / (HD / 2);
    const int per = (hi - lo + kGroups - 1) / kGroups, r0 = lo + group * per;
    const int r1 = min(r0 + per, hi);
    if (i < pairs && r0 < r1) {
      double s, c, ss = 0.0, sc = 1.0;
      sincospi(s_turns[i] * static_cast<double>(blk * kBlock + r0), &s, &c);
      if (r1 - r0 > 1) sincospi(s_turns[i], &ss, &sc);
      const int at = a.rope.type == PL_ROPE_LLAMA ? pair_place<true>(i, HD / 2)
                                                  : pair_place<false>(i, HD / 2);
      for (int r = r0; r < r1; ++r) {
        s_cs[r][at] = make_float2(static_cast<float>(c * a.rope.gain),
                                 static_cast<float>(s * a.rope.gain));
        const double nc = c * sc - s * ss;
        s = s * sc + c * ss;
        c = nc;
      }
    }
  }
  __syncthreads();
  // HD / 64 warps share a (head, K or V), so that no warp holds more than
  // 32 values a lane
  constexpr int kLanesPerRow = HD / 8, kRowsPerPass = 32 / kLanesPerRow;
  constexpr int kSplit = HD / 64, kRowsPerWarp = kBlock / kSplit;
  constexpr int kPasses = kRowsPerWarp / kRowsPerPass;
  constexpr int kTeams = kAppendThreads / 32 / kSplit;
  const int team = warp / kSplit, row_first = warp % kSplit * kRowsPerWarp;
  const int el = (lane % kLanesPerRow) * 8;
  const int sub = blk % kBlocksPerPage;
  int turn = 0;
  for (int u = team; u < 2 * a.g.n_kv_heads; u += kTeams) {
    const int h = u >> 1, kv = u & 1;
    const long long slab = a.g.slab(page, h, kv);
    uint8_t* dst = a.g.codes + (slab * kPage + sub * kBlock) * HD + el;
    float* sc = a.g.scales + slab * kBlocksPerPage + sub;
    const T* src = kv ? static_cast<const T*>(a.v) : static_cast<const T*>(a.k);
    const long long stride = kv ? a.v_stride : a.k_stride;
    const uint32_t old_bits = lo > 0 ? __float_as_uint(*sc) : 0u;
    float x[kPasses][8];
    float top = 0.f;
    uint32_t odd = 0;  // a NaN or infinity
    const int r_lane = row_first + lane / kLanesPerRow;
    const T* row_src = src + static_cast<long long>(e.tok0 + (blk * kBlock - row0) +
                                                    r_lane) * stride + h * HD;
    constexpr int kAhead = sizeof(T) == 4 ? 1 : 2;  // rows under way
#pragma unroll
    for (int p0 = 0; p0 < kPasses; p0 += kAhead) {
      Raw8<T> y[kAhead], z[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int r = (p0 + k) * kRowsPerPass + r_lane;
        if (r >= lo && r < hi)
          load_pair8(row_src + (p0 + k) * kRowsPerPass * stride, el, a.rope, kv == 0, y[k], z[k]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int p = p0 + k, r = p * kRowsPerPass + r_lane;
        unpack8(y[k], x[p]);
        if (r < lo || r >= hi) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[p][j] = 0.f;
        } else if (kv == 0) {
          float w[8];
          unpack8(z[k], w);
          rotate_pair8<HD>(el, a.rope, s_cs[r], x[p], w);
        }
#pragma unroll
        for (int j = 0; j < 8; j += 2) top = max3(top, fabsf(x[p][j]), fabsf(x[p][j + 1]));
        // x - x is 0 but for NaN and infinity
#pragma unroll
        for (int j = 0; j < 8; ++j) odd |= __float_as_uint(__fsub_rn(x[p][j], x[p][j]));
      }
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if (__any_sync(0xffffffffu, odd << 1)) top = __uint_as_float(0x7fc00000u);
    if constexpr (kSplit > 1) {
      if (lane == 0) s_top[turn][warp] = __float_as_uint(top);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * kSplit) : "memory");
#pragma unroll
      for (int w = 0; w < kSplit; ++w)
        top = __uint_as_float(max(__float_as_uint(top), s_top[turn][team * kSplit + w]));
      turn ^= 1;
    }
    float s = top;
    if (__float_as_uint(top) <= 0x7f800000u) s = __fdiv_rn(top, code_top<FMT>());
    s = __uint_as_float(max(__float_as_uint(s), old_bits));
    const float by = s > 0.f ? s : 1.f;
    const float inv = __fdiv_rn(1.f, by);
    const bool grown = lo > 0 && __float_as_uint(s) != old_bits;
    __syncwarp();  // every lane has read the old scale
    if (lane == 0 && row_first == 0) *sc = s;
    if (!(s < INFINITY)) {  // no code stands for a NaN: the scale alone says it
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[p][j] = 0.f;
    }
    if (by > 1e-25f && by < 1e25f) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[p][j] = quotient(x[p][j], by, inv);
    } else {
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          const float q = __fdiv_rn(x[p][0], by) + 0.f;  // in turn, to keep the code short
#pragma unroll
          for (int m = 0; m < 7; ++m) x[p][m] = x[p][m + 1];
          x[p][7] = q;
        }
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int r = p * kRowsPerPass + r_lane;
      if (r >= lo && r < hi)
        *reinterpret_cast<uint2*>(dst + r * HD) = encode8<FMT>(x[p]);
    }
    if (grown) {
      const float ratio = s > 0.f ? __fdiv_rn(__uint_as_float(old_bits), s) : 1.f;
#pragma unroll 1
      for (int r = r_lane; r < min(lo, row_first + kRowsPerWarp); r += kRowsPerPass) {
        uint2* at = reinterpret_cast<uint2*>(dst + r * HD);
        float y[8];
        decode8<FMT>(*at, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(y[j], ratio);
        *at = encode8<FMT>(y);
      }
    }
  }
}

// ---------------------------------------------------------------- read back
struct Kv8ReadArgs {
  Kv8Geo g;
  int n, total, max_rows;
  const int *seqs, *row0, *start;
  void *k, *v;
  long long k_stride, v_stride;
};

constexpr int kReadThreads = 256;

// Rows row0[i] .. of entry i, dequantised.  Grid (rows / 8 of the longest
// entry, entries); a warp per row.  Bound by HBM: 157 MB (8 x 4096 rows of 8
// heads of 128, e4m3 to BF16) in 33 us, 4.8 TB/s.
template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(
    const __grid_constant__ Kv8ReadArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Kv8Entry e;
  const bool ok = kv8_entry(a.g, blockIdx.y, a.total, a.max_rows, a.seqs, a.start, e);
  const int row0 = ok ? a.row0[blockIdx.y] : 0;
  if (!ok || row0 < 0 || row0 > e.len - e.n_tok) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    return;
  }
  const int j = blockIdx.x * (kReadThreads / 32) + warp;
  if (j >= e.n_tok) return;
  const int row = row0 + j;
  const int page = a.g.table[static_cast<long long>(e.slot) * a.g.max_pages + row / kPage];
  if (page < 0 || page >= a.g.n_pages) {
    if (lane == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    return;
  }
  const long long tok = e.tok0 + j;
  constexpr int kLanesPerRow = HD / 8;
  for (int u = lane; u < 2 * a.g.n_kv_heads * kLanesPerRow; u += 32) {
    const int el = (u % kLanesPerRow) * 8, hk = u / kLanesPerRow, h = hk >> 1, kv = hk & 1;
    const long long slab = a.g.slab(page, h, kv);
    const float s = a.g.scales[slab * kBlocksPerPage + row % kPage / kBlock];
    float x[8];
    decode8<FMT>(*reinterpret_cast<const uint2*>(
                     a.g.codes + (slab * kPage + row % kPage) * HD + el), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= s;
    T* dst = (kv ? static_cast<T*>(a.v) + tok * a.v_stride : static_cast<T*>(a.k) + tok * a.k_stride) +
             h * HD + el;
    store8(dst, x);
  }
}

// ---------------------------------------------------------------- pages
// The books (table, lens, refs) live on the device, so that a step that
// grows sequences can be captured in a CUDA graph.  One block of 1024
// threads changes them (kv8_plan_kernel) and leaves the list of pages to
// copy in the workspace; kv8_move_kernel, queued behind it with
// programmatic dependent launch, copies them with the whole GPU.  Pages
// are granted lowest index first, in the order of the call's list, so the
// same calls give the same tables.
constexpr int kPlanThreads = 1024;
constexpr int kPlanSeqs = 1024;  // entries per call

enum { PLAN_RESIZE = 0, PLAN_FORK = 1, PLAN_COMPACT = 2, PLAN_COPY = 3 };

struct Kv8PlanArgs {
  Kv8Geo g;
  int op, n;
  const int *a, *b;     // resize: slots, rows (nullptr: 0); fork: src, dst slots; copy: src, dst pages
  int *src, *dst;       // [n_pages] pages to copy
  int* mark;            // [n_pages] free pages (resize), new place of a page (compact), marks (copy)
};

// Exclusive prefix sum of `v` over the block; the sum of all in `total`.
template <typename N>
__device__ __forceinline__ N block_scan(N v, N& total, long long* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // s_warp may still be read from an earlier scan
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    N w = static_cast<N>(s_warp[lane]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const N y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = static_cast<N>(s_warp[31]);
  return x - v + (warp ? static_cast<N>(s_warp[warp - 1]) : 0);
}

__device__ __forceinline__ int pages_of(int rows) { return (rows + kPage - 1) / kPage; }

__device__ void plan_resize(const Kv8PlanArgs& a, long long* s_warp, int (*s_e)[kPlanSeqs]) {
  const Kv8Geo& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* s_slot = s_e[0];
  int* s_old = s_e[1];
  int* s_new = s_e[2];
  int* s_tail = s_e[3];   // shared last page of a growing entry, else -1
  int* s_off = s_e[4];    // first granted page (bit 31: the first one replaces the tail)
  bool bad = false;
  if (tid < a.n) {
    const int slot = a.a[tid], want = a.b ? a.b[tid] : 0;
    s_slot[tid] = slot;
    bad = slot < 0 || slot >= g.n_seqs || want < 0 || want > g.max_pages * kPage;
    const int have = bad ? 0 : g.lens[slot];
    bad |= have < 0 || have > g.max_pages * kPage;
    s_old[tid] = have;
    s_new[tid] = want;
    int tail = -1;
    if (!bad && want > have && have % kPage) {
      tail = g.table[static_cast<long long>(slot) * g.max_pages + have / kPage];
      bad |= tail < 0 || tail >= g.n_pages;
    }
    s_tail[tid] = tail;
  }
  __syncthreads();
  if (tid < a.n)
    for (int j = 0; j < tid; ++j) bad |= s_slot[j] == s_slot[tid];
  if (__syncthreads_or(bad)) {
    if (tid == 0) atomicOr(&g.head->err, ERR_BAD_ARG);
    return;
  }
  // pages given up come first, so that the same call may grant them again
  for (int i = warp; i < a.n; i += kPlanThreads / 32) {
    const int* row = g.table + static_cast<long long>(s_slot[i]) * g.max_pages;
    for (int j = pages_of(s_new[i]) + lane; j < pages_of(s_old[i]); j += 32) {
      const int p = row[j];
      if (p >= 0 && p < g.n_pages) atomicSub(&g.refs[p], 1);
    }
  }
  __syncthreads();
  // an entry that grows within a page it shares takes a copy of it; the
  // last sharer of the call keeps the page if nobody else holds it
  long long need = 0;  // 1024 entries of up to 2^25 pages
  int copy = 0;
  if (tid < a.n) {
    const int tail = s_tail[tid];
    if (tail >= 0) {
      int rank = 0;
      for (int j = 0; j < tid; ++j) rank += s_tail[j] == tail;
      copy = __ldcg(&g.refs[tail]) - rank > 1;
    }
    need = max(0, pages_of(s_new[tid]) - pages_of(s_old[tid])) + copy;
  }
  long long wanted;
  int n_copies;
  const long long off_wide = block_scan(need, wanted, s_warp);
  const int copy_at = block_scan(copy, n_copies, s_warp);
  // the lowest free pages, in order (each thread a contiguous run of pages)
  const int per = (g.n_pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(tid * per, g.n_pages), p1 = min(p0 + per, g.n_pages);
  int free_here = 0;
  for (int p = p0; p < p1; ++p) free_here += __ldcg(&g.refs[p]) == 0;
  int n_free;
  int at = block_scan(free_here, n_free, s_warp);
  if (wanted > n_free) {  // nothing is changed: the released pages are taken back
    for (int i = warp; i < a.n; i += kPlanThreads / 32) {
      const int* row = g.table + static_cast<long long>(s_slot[i]) * g.max_pages;
      for (int j = pages_of(s_new[i]) + lane; j < pages_of(s_old[i]); j += 32) {
        const int p = row[j];
        if (p >= 0 && p < g.n_pages) atomicAdd(&g.refs[p], 1);
      }
    }
    if (tid == 0) atomicOr(&g.head->err, ERR_NO_PAGES);
    return;
  }
  // from here on no more than the pool's pages, fewer than 2^30
  const int total = static_cast<int>(wanted), off = static_cast<int>(off_wide);
  for (int p = p0; p < p1 && at < total; ++p)
    if (__ldcg(&g.refs[p]) == 0) a.mark[at++] = p;
  if (tid < a.n) s_off[tid] = off | (copy << 31);
  __syncthreads();
  if (tid < a.n && copy) {
    const int to = a.mark[off];
    a.src[copy_at] = s_tail[tid];
    a.dst[copy_at] = to;
    atomicSub(&g.refs[s_tail[tid]], 1);
    g.table[static_cast<long long>(s_slot[tid]) * g.max_pages + s_old[tid] / kPage] = to;
  }
  for (int i = tid; i < total; i += kPlanThreads) g.refs[a.mark[i]] = 1;
  for (int i = warp; i < a.n; i += kPlanThreads / 32) {
    int* row = g.table + static_cast<long long>(s_slot[i]) * g.max_pages;
    const int had = pages_of(s_old[i]), has = pages_of(s_new[i]);
    const int first = (s_off[i] & 0x7fffffff) + (s_off[i] < 0 ? 1 : 0);
    for (int j = had + lane; j < has; j += 32) row[j] = a.mark[first + j - had];
    for (int j = has + lane; j < had; j += 32) row[j] = -1;
    if (lane == 0) g.lens[s_slot[i]] = s_new[i];
  }
  if (tid == 0) g.head->n_copies = n_copies;
}

__device__ void plan_fork(const Kv8PlanArgs& a, int (*s_e)[kPlanSeqs]) {
  const Kv8Geo& g = a.g;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* s_src = s_e[0];
  int* s_dst = s_e[1];
  bool bad = false;
  if (tid < a.n) {
    s_src[tid] = a.a[tid];
    s_dst[tid] = a.b[tid];
    bad = s_src[tid] < 0 || s_src[tid] >= g.n_seqs || s_dst[tid] < 0 || s_dst[tid] >= g.n_seqs;
    if (!bad)
      bad = g.lens[s_src[tid]] < 0 || g.lens[s_src[tid]] > g.max_pages * kPage ||
            g.lens[s_dst[tid]] < 0 || g.lens[s_dst[tid]] > g.max_pages * kPage;
  }
  __syncthreads();
  if (tid < a.n)
    for (int j = 0; j < a.n; ++j) {
      bad |= j < tid && s_dst[j] == s_dst[tid];
      bad |= s_src[j] == s_dst[tid];
    }
  if (__syncthreads_or(bad)) {
    if (tid == 0) atomicOr(&g.head->err, ERR_BAD_ARG);
    return;
  }
  for (int i = warp; i < a.n; i += kPlanThreads / 32) {
    const int* from = g.table + static_cast<long long>(s_src[i]) * g.max_pages;
    int* to = g.table + static_cast<long long>(s_dst[i]) * g.max_pages;
    const int rows = g.lens[s_src[i]], had = pages_of(g.lens[s_dst[i]]), has = pages_of(rows);
    for (int j = lane; j < max(had, has); j += 32) {
      if (j < had) {
        const int p = to[j];
        if (p >= 0 && p < g.n_pages) atomicSub(&g.refs[p], 1);
      }
      const int p = j < has ? from[j] : -1;
      to[j] = p;
      if (p >= 0 && p < g.n_pages) atomicAdd(&g.refs[p], 1);
    }
    __syncwarp();
    if (lane == 0) g.lens[s_dst[i]] = rows;
  }
}

__device__ void plan_compact(const Kv8PlanArgs& a, long long* s_warp) {
  const Kv8Geo& g = a.g;
  const int tid = threadIdx.x;
  const int per = (g.n_pages + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(tid * per, g.n_pages), p1 = min(p0 + per, g.n_pages);
  int used_here = 0, used, n_holes, n_moves;
  for (int p = p0; p < p1; ++p) used_here += g.refs[p] != 0;
  block_scan(used_here, used, s_warp);
  int holes = 0, moves = 0;
  for (int p = p0; p < p1; ++p) {
    const bool in_use = g.refs[p] != 0;
    holes += !in_use && p < used;
    moves += in_use && p >= used;
  }
  int hole_at = block_scan(holes, n_holes, s_warp);
  int move_at = block_scan(moves, n_moves, s_warp);
  for (int p = p0; p < p1; ++p) {
    const bool in_use = g.refs[p] != 0;
    a.mark[p] = p;
    if (!in_use && p < used) a.dst[hole_at++] = p;
    if (in_use && p >= used) a.src[move_at++] = p;
  }
  __syncthreads();
  for (int i = tid; i < n_moves; i += kPlanThreads) {
    const int from = a.src[i], to = a.dst[i];
    a.mark[from] = to;
    g.refs[to] = g.refs[from];
    g.refs[from] = 0;
  }
  if (tid == 0) g.head->n_copies = n_moves;
}

__device__ void plan_copy(const Kv8PlanArgs& a) {
  const Kv8Geo& g = a.g;
  const int tid = threadIdx.x;
  bool bad = false;
  for (int i = tid; i < a.n; i += kPlanThreads)
    bad |= a.a[i] < 0 || a.a[i] >= g.n_pages || a.b[i] < 0 || a.b[i] >= g.n_pages;
  if (!__syncthreads_or(bad)) {
    // a page written twice, or read and written, has no defined result
    for (int i = tid; i < a.n; i += kPlanThreads) a.mark[a.a[i]] = a.mark[a.b[i]] = 0;
    __syncthreads();
    for (int i = tid; i < a.n; i += kPlanThreads)
      if (atomicAdd(&a.mark[a.b[i]], 1) != 0) bad = true;
    __syncthreads();
    for (int i = tid; i < a.n; i += kPlanThreads) bad |= __ldcg(&a.mark[a.a[i]]) != 0;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) atomicOr(&g.head->err, ERR_BAD_ARG);
    return;
  }
  for (int i = tid; i < a.n; i += kPlanThreads) {
    a.src[i] = a.a[i];
    a.dst[i] = a.b[i];
  }
  if (tid == 0) g.head->n_copies = a.n;
}

__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(
    const __grid_constant__ Kv8PlanArgs a) {
  __shared__ long long s_warp[32];
  __shared__ int s_e[5][kPlanSeqs];
  // the copies may become resident now; they wait for this grid's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) a.g.head->n_copies = 0;
  __syncthreads();
  if (a.op == PLAN_RESIZE) plan_resize(a, s_warp, s_e);
  else if (a.op == PLAN_FORK) plan_fork(a, s_e);
  else if (a.op == PLAN_COMPACT) plan_compact(a, s_warp);
  else plan_copy(a);
}

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;
constexpr int kMoveChunk = kMoveThreads * kMoveUnroll * 16;  // bytes per step of a block

// Copies the listed pages (codes in chunks of 32 KB, then the scales), and
// after a compaction (`remap`) sends the table to the new places.  Bound by
// HBM: a page is read and written once (compacting 365 MB over 22 layers: 57
// us, 6.4 TB/s, as a plain copy; the books before it 6.5 us).
__global__ void __launch_bounds__(kMoveThreads) kv8_move_kernel(
    const __grid_constant__ Kv8Geo g, const int* src, const int* dst, const int* mark, int remap,
    long long code_bytes, long long scale_bytes) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long n = __ldcg(&g.head->n_copies);
  const int per_page = static_cast<int>((code_bytes + kMoveChunk - 1) / kMoveChunk) +
                       static_cast<int>((scale_bytes + kMoveChunk - 1) / kMoveChunk);
  const int code_chunks = static_cast<int>((code_bytes + kMoveChunk - 1) / kMoveChunk);
  for (long long u = blockIdx.x; u < n * per_page; u += gridDim.x) {
    const int i = static_cast<int>(u / per_page), c = static_cast<int>(u % per_page);
    const bool codes = c < code_chunks;
    const long long bytes = codes ? code_bytes : scale_bytes;
    const long long at = static_cast<long long>(codes ? c : c - code_chunks) * kMoveChunk;
    const uint8_t* base = codes ? g.codes : reinterpret_cast<const uint8_t*>(g.scales);
    const uint8_t* from = base + __ldcg(src + i) * bytes + at;
    uint8_t* to = const_cast<uint8_t*>(base) + __ldcg(dst + i) * bytes + at;
    uint4 v[kMoveUnroll];
#pragma unroll
    for (int k = 0; k < kMoveUnroll; ++k) {
      const long long o = (static_cast<long long>(k) * kMoveThreads + threadIdx.x) * 16;
      if (at + o < bytes) v[k] = __ldcs(reinterpret_cast<const uint4*>(from + o));
    }
#pragma unroll
    for (int k = 0; k < kMoveUnroll; ++k) {
      const long long o = (static_cast<long long>(k) * kMoveThreads + threadIdx.x) * 16;
      if (at + o < bytes) __stcs(reinterpret_cast<uint4*>(to + o), v[k]);
    }
  }
  if (!remap || n == 0) return;
  // pages at and above the number in use have moved: refs is 0 there now
  const long long cells = static_cast<long long>(g.n_seqs) * g.max_pages;
  for (long long t = static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x; t < cells;
       t += static_cast<long long>(gridDim.x) * kMoveThreads) {
    const int p = g.table[t];
    if (p >= 0 && p < g.n_pages && g.refs[p] == 0) g.table[t] = mark[p];
  }
}

}  // namespace pl
