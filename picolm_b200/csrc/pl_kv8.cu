// pl_kv8.cu -- the entry points of the rotary operator and of the 8-bit
// paged KV cache (include/pl_attn.h): argument checks and dispatch.  They
// hold no state: everything a call needs is in its pl_rope or pl_kv8.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../include/pl_attn.h"
#include "kern_kv8.cuh"
#include "kern_kv8_attn.cuh"
#include "kern_kv8_chunk.cuh"
#include "kern_rope.cuh"
#include "pl_kv8.h"

namespace pl_module {

cudaError_t kv8_wait_limit(uint64_t ns) {
  return cudaMemcpyToSymbol(pl::g_wait_limit_ns, &ns, sizeof(ns));
}

}  // namespace pl_module

namespace {

#define PL_CUDA(call)                                                     \
  do {                                                                    \
    cudaError_t e_ = (call);                                              \
    if (e_ != cudaSuccess) {                                              \
      std::fprintf(stderr, "pl_attn: %s failed: %s (%s:%d)\n", #call,      \
                   cudaGetErrorString(e_), __FILE__, __LINE__);           \
      return PL_ECUDA;                                                    \
    }                                                                     \
  } while (0)

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

size_t elem_size(int dtype) { return dtype == PL_F32 ? 4 : 2; }

bool good_dtype(int dtype) { return dtype == PL_F32 || dtype == PL_F16 || dtype == PL_BF16; }

// Launch behind the kernel queued before it on the stream, with
// programmatic dependent launch where the kernel waits for it itself.
template <typename... P, typename... A>
int launch(void (*kern)(P...), dim3 grid, int threads, int smem, void* stream, bool overlap,
           A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  PL_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
  return PL_OK;
}

// SM count of the current device (0: no usable device), looked up once.
int sm_count() {
  static int cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && cached[dev]) return cached[dev];
  int major = 0, n = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      major != 10 ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  if (dev < 64) cached[dev] = n;
  return n;
}

// Blocks of an attention grid, at most (the workspace holds two
// partials for each).
constexpr int kMaxBlocks = 160;

// Shared memory above 48 KB is an attribute of a kernel on each device: set
// the first time this kernel launches there.  With regs, the kernel's
// warpgroups share out exactly that many registers a thread (setmaxnreg): from
// a smaller allocation an increase would wait for good, so another count is
// refused.
template <typename K>
int allow_smem(K kern, int bytes, std::atomic<unsigned long long>& done, int regs = 0) {
  int dev = 0;
  PL_CUDA(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return PL_OK;
  PL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (regs) {
    cudaFuncAttributes at;
    PL_CUDA(cudaFuncGetAttributes(&at, kern));
    if (at.numRegs != regs) {
      std::fprintf(stderr, "pl_attn: a kernel has %d registers a thread instead of %d\n",
                   at.numRegs, regs);
      return PL_EFAIL;
    }
  }
  done.fetch_or(bit, std::memory_order_release);
  return PL_OK;
}

// The codes as [slab][64 rows][head_dim] bytes, slab = (page, layer, head,
// K or V), read in boxes of `rows` rows of K and V under the swizzle of a
// row's width.
int codes_map(const pl_kv8* c, int rows, CUtensorMap* m) {
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                               const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<EncodeFn> encode{nullptr};
  EncodeFn fn = encode.load(std::memory_order_acquire);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) !=
            cudaSuccess ||
        res != cudaDriverEntryPointSuccess || !p)
      return PL_ECUDA;
    fn = reinterpret_cast<EncodeFn>(p);
    encode.store(fn, std::memory_order_release);
  }
  const cuuint64_t hd = static_cast<cuuint64_t>(c->head_dim);
  const cuuint64_t dims[3] = {
      hd, PL_KV8_PAGE,
      static_cast<cuuint64_t>(c->n_pages) * c->n_layers * c->n_kv_heads * 2};
  const cuuint64_t strides[2] = {hd, hd * PL_KV8_PAGE};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(hd), static_cast<cuuint32_t>(rows), 2u};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c->codes, dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE,
         c->head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    std::fprintf(stderr, "pl_attn: cuTensorMapEncodeTiled failed (%d)\n", static_cast<int>(r));
    return PL_ECUDA;
  }
  return PL_OK;
}

// ------------------------------------------------------------ cache checks
int check_kv8_shape(const pl_kv8* c) {
  if (!c) return PL_EARG;
  if (c->n_layers <= 0 || c->n_heads <= 0 || c->n_kv_heads <= 0 || c->n_pages <= 0 ||
      c->n_seqs <= 0 || c->max_pages <= 0 || c->max_pages > INT32_MAX / PL_KV8_PAGE ||
      c->device < 0)
    return PL_EARG;
  if (c->format != PL_KV8_INT8 && c->format != PL_KV8_E4M3) return PL_EARG;
  if (c->head_dim != 64 && c->head_dim != 128) return PL_EUNSUPPORTED;
  if (c->n_heads % c->n_kv_heads || c->n_heads / c->n_kv_heads > pl::kKv8MaxGroup ||
      c->n_kv_heads > 1024)
    return PL_EUNSUPPORTED;
  // (page, layer, head, K or V) is a 31-bit coordinate of the bulk copies
  if (static_cast<double>(c->n_pages) * c->n_layers * c->n_kv_heads * 2 > 2147483647.0)
    return PL_EUNSUPPORTED;
  if (c->rope.dim < 0 || (c->rope.dim & 1) || c->rope.dim > c->head_dim ||
      (c->rope.dim && (c->rope.head_dim != c->head_dim ||
                       (c->rope.type != PL_ROPE_LLAMA && c->rope.type != PL_ROPE_QWEN))))
    return PL_EARG;
  return PL_OK;
}

size_t plan_bytes(const pl_kv8* c) {  // src, dst, mark: one int a page each
  return (static_cast<size_t>(c->n_pages) * 4 + 255) / 256 * 256 * 3;
}

// Attention: two partials a block (of two 128-row tiles, or of one token's
// heads, which are smaller), then an arrival counter for each block.
size_t part_bytes(const pl_kv8* c) {
  return static_cast<size_t>(2) * kMaxBlocks * 2 * pl::kChRows * (c->head_dim + 2) * 4;
}
// FP32 sums of the chunk attention's output tiles, one pair of tiles a block.
size_t sum_bytes(const pl_kv8* c) {
  return static_cast<size_t>(kMaxBlocks) * 2 * pl::kChRows * c->head_dim * 4;
}
size_t arrive_bytes(const pl_kv8*) { return static_cast<size_t>(kMaxBlocks) * 4; }

size_t work_bytes(const pl_kv8* c) {
  return sizeof(pl::Kv8Head) + plan_bytes(c) + part_bytes(c) + sum_bytes(c) + arrive_bytes(c);
}

float* work_part(const pl_kv8* c) {
  return reinterpret_cast<float*>(static_cast<uint8_t*>(c->work) + sizeof(pl::Kv8Head) +
                                  plan_bytes(c));
}
float* work_sums(const pl_kv8* c) { return work_part(c) + part_bytes(c) / 4; }
int* work_arrived(const pl_kv8* c) {
  return reinterpret_cast<int*>(work_sums(c) + sum_bytes(c) / 4);
}

// Every call on a cache: its shape, its memory and the current device.
int check_kv8(const pl_kv8* c) {
  const int rc = check_kv8_shape(c);
  if (rc) return rc;
  if (!c->codes || !c->scales || !c->table || !c->lens || !c->refs || !c->work ||
      !aligned(c->codes, 256) || !aligned(c->scales, 256) || !aligned(c->work, 256) ||
      !aligned(c->table, 4) || !aligned(c->lens, 4) || !aligned(c->refs, 4) ||
      c->work_bytes < work_bytes(c))
    return PL_EARG;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev != c->device || !sm_count()) return PL_EDEVICE;
  return PL_OK;
}

pl::Kv8Geo geo(const pl_kv8* c, int layer) {
  pl::Kv8Geo g;
  g.codes = static_cast<uint8_t*>(c->codes);
  g.scales = c->scales;
  g.table = c->table;
  g.lens = c->lens;
  g.refs = c->refs;
  g.head = static_cast<pl::Kv8Head*>(c->work);
  g.n_layers = c->n_layers;
  g.n_kv_heads = c->n_kv_heads;
  g.n_pages = c->n_pages;
  g.n_seqs = c->n_seqs;
  g.max_pages = c->max_pages;
  g.layer = layer;
  return g;
}

// A ragged call: entries, tokens, layer.  PL_OK with *none set when there is
// nothing to do.
int check_call(const pl_kv8* c, int layer, int n, const void* d_seqs, const void* d_start,
               int total, int max_tok, int dtype, bool* none) {
  const int rc = check_kv8(c);
  if (rc) return rc;
  if (layer < 0 || layer >= c->n_layers || n < 0 || n > pl::kPlanSeqs || total < 0 ||
      max_tok < 0 || max_tok > c->max_pages * PL_KV8_PAGE || !good_dtype(dtype))
    return PL_EARG;
  if (!d_start && (total != n || max_tok != 1)) return PL_EARG;
  // tiles of a call are counted in 31 bits
  if (static_cast<long long>(n) * c->max_pages * c->n_kv_heads * 4 > INT32_MAX) return PL_EARG;
  *none = n == 0 || total == 0 || max_tok == 0;
  if (!*none && !d_seqs) return PL_EARG;
  return PL_OK;
}

bool good_rows(const void* p, long long stride, int heads, int head_dim, int dtype) {
  return p && aligned(p, 16) && stride >= static_cast<long long>(heads) * head_dim &&
         stride * static_cast<long long>(elem_size(dtype)) % 16 == 0;
}

// f<T, HD, FMT> by the run-time types of a call.
template <template <typename, int, int> class F, typename T, typename... A>
int by_shape(const pl_kv8* c, A... a) {
  if (c->head_dim == 64)
    return c->format == PL_KV8_INT8 ? F<T, 64, PL_KV8_INT8>::run(c, a...)
                                    : F<T, 64, PL_KV8_E4M3>::run(c, a...);
  return c->format == PL_KV8_INT8 ? F<T, 128, PL_KV8_INT8>::run(c, a...)
                                  : F<T, 128, PL_KV8_E4M3>::run(c, a...);
}
template <template <typename, int, int> class F, typename... A>
int by_type(const pl_kv8* c, int dtype, A... a) {
  if (dtype == PL_F32) return by_shape<F, float>(c, a...);
  if (dtype == PL_F16) return by_shape<F, __half>(c, a...);
  return by_shape<F, __nv_bfloat16>(c, a...);
}

template <typename T, int HD, int FMT>
struct Append {
  static int run(const pl_kv8*, const pl::Kv8AppendArgs& a, void* st) {
    const int blocks = (a.max_tok + PL_KV8_BLOCK - 2) / PL_KV8_BLOCK + 1;
    return launch(pl::kv8_append_kernel<T, HD, FMT>, dim3(blocks, a.n), pl::kAppendThreads, 0, st,
                  true, a);
  }
};

template <typename T, int HD, int FMT>
struct Read {
  static int run(const pl_kv8*, const pl::Kv8ReadArgs& a, void* st) {
    const int per = pl::kReadThreads / 32;
    return launch(pl::kv8_read_kernel<T, HD, FMT>, dim3((a.max_rows + per - 1) / per, a.n),
                  pl::kReadThreads, 0, st, false, a);
  }
};

// One token an entry; with k and v, they are appended by the same launch.
template <typename T, int HD, int FMT, bool APPEND>
int run_decode(const pl_kv8* c, pl::Kv8DecodeArgs d, void* st) {
  d.part = work_part(c);
  d.arrived = work_arrived(c);
  CUtensorMap tm;
  int rc = codes_map(c, pl::DecShape<HD>::kTileRows, &tm);
  if (rc) return rc;
  constexpr int smem = static_cast<int>(sizeof(pl::DecSmem<HD>)) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of the one-token attention");
  static std::atomic<unsigned long long> done{0};
  auto kern = pl::kv8_decode_kernel<T, HD, FMT, APPEND>;
  if ((rc = allow_smem(kern, smem, done))) return rc;
  const int blocks = sm_count() < kMaxBlocks ? sm_count() : kMaxBlocks;
  return launch(kern, dim3(blocks), pl::DecShape<HD>::kThreads, smem, st, true, d, tm);
}

template <typename T, int HD, int FMT>
struct Attend {
  static int run(const pl_kv8* c, const pl::Kv8AttnArgs& a, void* st) {
    if (a.max_tok == 1) {
      pl::Kv8DecodeArgs d = {};
      d.a = a;
      return run_decode<T, HD, FMT, false>(c, d, st);
    }
    constexpr int PARTS = pl::ch_parts<T>();
    constexpr int smem = static_cast<int>(sizeof(pl::ChSmem<HD, PARTS>)) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of the chunk attention");
    static std::atomic<unsigned long long> done{0};
    auto kern = pl::kv8_chunk_kernel<T, HD, FMT>;
    pl::Kv8ChunkArgs ch = {};
    ch.a = a;
    ch.part = work_part(c);
    ch.sums = work_sums(c);
    ch.arrived = work_arrived(c);
    const int rc = allow_smem(kern, smem, done, pl::kChLaunchRegs);
    if (rc) return rc;
    const int blocks = sm_count() < kMaxBlocks ? sm_count() : kMaxBlocks;
    return launch(kern, dim3(blocks), pl::kChThreads, smem, st, true, ch);
  }
};

template <typename T, int HD, int FMT>
struct Decode {
  static int run(const pl_kv8* c, const pl::Kv8DecodeArgs& d, void* st) {
    return run_decode<T, HD, FMT, true>(c, d, st);
  }
};

pl::Kv8AttnArgs attn_args(const pl_kv8* c, int layer, int n, const int* d_seqs, const int* d_start,
                          int total, int max_tok, const void* d_q, long long q_stride, void* d_out,
                          long long out_stride) {
  pl::Kv8AttnArgs a;
  a.g = geo(c, layer);
  a.rope = c->rope;
  a.n = n;
  a.total = total;
  a.max_tok = max_tok;
  a.n_heads = c->n_heads;
  a.group = c->n_heads / c->n_kv_heads;
  a.seqs = d_seqs;
  a.start = d_start;
  a.q = d_q;
  a.out = d_out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.score_scale = static_cast<float>(1.4426950408889634 / std::sqrt(double(c->head_dim)));
  return a;
}

int plan(const pl_kv8* c, int op, int n, const int* a, const int* b, bool moves, void* stream) {
  pl::Kv8PlanArgs p;
  p.g = geo(c, 0);
  p.op = op;
  p.n = n;
  p.a = a;
  p.b = b;
  const size_t each = plan_bytes(c) / 3;
  uint8_t* w = static_cast<uint8_t*>(c->work) + sizeof(pl::Kv8Head);
  p.src = reinterpret_cast<int*>(w);
  p.dst = reinterpret_cast<int*>(w + each);
  p.mark = reinterpret_cast<int*>(w + 2 * each);
  int rc = launch(pl::kv8_plan_kernel, dim3(1), pl::kPlanThreads, 0, stream, false, p);
  if (rc || !moves) return rc;
  const long long slabs = static_cast<long long>(c->n_layers) * c->n_kv_heads * 2;
  const long long code_bytes = slabs * PL_KV8_PAGE * c->head_dim;
  const long long scale_bytes = slabs * pl::kBlocksPerPage * 4;
  return launch(pl::kv8_move_kernel, dim3(sm_count() * 8), pl::kMoveThreads, 0, stream, true, p.g,
                p.src, p.dst, p.mark, op == pl::PLAN_COMPACT ? 1 : 0, code_bytes, scale_bytes);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------ rotary
int pl_rope_init(pl_rope* r, int type, int head_dim, int dim, double base, int scaling,
                 double factor, int orig_len, double low, double high) {
  if (!r || (type != PL_ROPE_LLAMA && type != PL_ROPE_QWEN)) return PL_EARG;
  if (head_dim < 8 || head_dim > 2 * PL_ROPE_MAX_PAIRS || head_dim % 8) return PL_EUNSUPPORTED;
  if (dim < 0 || dim > head_dim || (dim & 1) || !(base > 0.0) || !std::isfinite(base))
    return PL_EARG;
  if (scaling < PL_ROPE_SCALE_NONE || scaling > PL_ROPE_SCALE_LLAMA3) return PL_EARG;
  if (scaling != PL_ROPE_SCALE_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return PL_EARG;
  if (scaling >= PL_ROPE_SCALE_YARN &&
      (orig_len <= 0 || !(low > 0.0) || !(high > low) || !std::isfinite(high) || base == 1.0))
    return PL_EARG;
  std::memset(r, 0, sizeof(*r));
  r->type = type;
  r->head_dim = head_dim;
  r->dim = dim;
  r->gain = scaling == PL_ROPE_SCALE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
  const double pi = 3.14159265358979323846;
  double first = 0.0, last = 1.0;
  if (scaling == PL_ROPE_SCALE_YARN) {
    // the (fractional) pair that turns `turns` times in orig_len positions
    auto pair_of = [&](double turns) {
      return dim * std::log(orig_len / (turns * 2.0 * pi)) / (2.0 * std::log(base));
    };
    first = std::fmax(std::floor(pair_of(high)), 0.0);
    last = std::fmin(std::ceil(pair_of(low)), dim - 1.0);
  }
  for (int i = 0; i < dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / dim);
    if (scaling == PL_ROPE_SCALE_LINEAR) {
      f /= factor;
    } else if (scaling == PL_ROPE_SCALE_YARN) {
      const double part =
          std::fmin(std::fmax((i - first) / std::fmax(last - first, 0.001), 0.0), 1.0);
      f = f / factor * part + f * (1.0 - part);
    } else if (scaling == PL_ROPE_SCALE_LLAMA3) {
      const double turns = orig_len * f / (2.0 * pi);
      const double keep = std::fmin(std::fmax((turns - low) / (high - low), 0.0), 1.0);
      f *= (1.0 - keep) / factor + keep;
    }
    r->half_turns[i] = f / pi;
  }
  return PL_OK;
}

int pl_rope_rows_dev(const pl_rope* r, int dtype, int n, const int* d_pos, int n_heads,
                     const void* d_q, long long q_stride, void* d_q_out, long long q_out_stride,
                     int n_kv_heads, const void* d_k, long long k_stride, void* d_k_out,
                     long long k_out_stride, int adjoint, void* stream) {
  if (!r || !good_dtype(dtype) || n < 0 || n_heads < 0 || n_kv_heads < 0 ||
      n_heads > 65536 || n_kv_heads > 65536 || r->head_dim < 8 ||
      r->head_dim > 2 * PL_ROPE_MAX_PAIRS || r->head_dim % 8 || r->dim < 0 ||
      r->dim > r->head_dim || (r->dim & 1) ||
      (r->type != PL_ROPE_LLAMA && r->type != PL_ROPE_QWEN))
    return PL_EARG;
  if (n == 0 || n_heads + n_kv_heads == 0) return PL_OK;
  const size_t es = elem_size(dtype);
  auto bad = [&](int heads, const void* p, long long s, const void* o, long long os) {
    const long long w = static_cast<long long>(heads) * r->head_dim;
    return heads && (!p || !o || s < w || os < w || !aligned(p, es) || !aligned(o, es));
  };
  if (!d_pos || bad(n_heads, d_q, q_stride, d_q_out, q_out_stride) ||
      bad(n_kv_heads, d_k, k_stride, d_k_out, k_out_stride))
    return PL_EARG;
  const int sms = sm_count();
  if (!sms) return PL_EDEVICE;
  pl::RopeRowsArgs a;
  a.rope = *r;
  a.pos = d_pos;
  a.n = n;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.adjoint = adjoint;
  a.q = d_q;
  a.k = d_k;
  a.qo = d_q_out;
  a.ko = d_k_out;
  a.q_stride = q_stride;
  a.qo_stride = q_out_stride;
  a.k_stride = k_stride;
  a.ko_stride = k_out_stride;
  // as many rows a block as leave every SM a few blocks
  const int rows = n / (4 * sms);
  a.rows_per_block = rows < 1 ? 1 : rows > pl::kRopeRows ? pl::kRopeRows : rows;
  const dim3 grid((n + a.rows_per_block - 1) / a.rows_per_block);
  const int half = r->dim / 2;
  const bool llama = r->type == PL_ROPE_LLAMA;
  auto vec = [&](int heads, const void* p, long long s, const void* o, long long os) {
    const long long e = static_cast<long long>(es);
    return !heads || (aligned(p, 16) && aligned(o, 16) && s * e % 16 == 0 && os * e % 16 == 0);
  };
  const bool fast = (llama || half % 8 == 0) &&
                    vec(n_heads, d_q, q_stride, d_q_out, q_out_stride) &&
                    vec(n_kv_heads, d_k, k_stride, d_k_out, k_out_stride);
  a.per_head = llama ? r->head_dim / 8 : half / 8 + (r->head_dim - r->dim) / 8;
  a.units = a.per_head * (n_heads + n_kv_heads);
  a.per_head_inv = fast ? ((1ull << 32) + a.per_head - 1) / a.per_head : 0;
  // blocks of equal width along a row
  const int across = (a.units + pl::kRopeThreads - 1) / pl::kRopeThreads;
  const int width = fast ? ((a.units + across - 1) / across + 31) / 32 * 32 : pl::kRopeThreads;
  const dim3 grid_vec(grid.x, across);
  auto go = [&](auto any, auto by_pairs, auto by_halves) {
    return launch(!fast ? any : llama ? by_pairs : by_halves, fast ? grid_vec : grid,
                  width, 0, stream, false, a);
  };
  if (dtype == PL_F32)
    return go(pl::rope_rows_any_kernel<float>, pl::rope_rows_kernel<float, true>,
              pl::rope_rows_kernel<float, false>);
  if (dtype == PL_F16)
    return go(pl::rope_rows_any_kernel<__half>, pl::rope_rows_kernel<__half, true>,
              pl::rope_rows_kernel<__half, false>);
  return go(pl::rope_rows_any_kernel<__nv_bfloat16>, pl::rope_rows_kernel<__nv_bfloat16, true>,
            pl::rope_rows_kernel<__nv_bfloat16, false>);
}

// ------------------------------------------------------------------- cache
int pl_kv8_work_bytes(const pl_kv8* c, size_t* bytes) {
  const int rc = check_kv8_shape(c);
  if (rc) return rc;
  if (!bytes) return PL_EARG;
  *bytes = work_bytes(c);
  return PL_OK;
}

int pl_kv8_alloc(pl_kv8* c) {
  const int rc = check_kv8_shape(c);
  if (rc) return rc;
  int dev = -1, count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || c->device >= count) return PL_EDEVICE;
  if (cudaGetDevice(&dev) != cudaSuccess || dev != c->device || !sm_count()) return PL_EDEVICE;
  const size_t slabs = static_cast<size_t>(c->n_pages) * c->n_layers * c->n_kv_heads * 2;
  const size_t cells = static_cast<size_t>(c->n_seqs) * c->max_pages;
  struct {
    void** p;
    size_t bytes;
    int fill;
  } const want[] = {
      {&c->codes, slabs * PL_KV8_PAGE * c->head_dim, 0},
      {reinterpret_cast<void**>(&c->scales), slabs * pl::kBlocksPerPage * 4, 0},
      {reinterpret_cast<void**>(&c->table), cells * 4, 0xff},
      {reinterpret_cast<void**>(&c->lens), static_cast<size_t>(c->n_seqs) * 4, 0},
      {reinterpret_cast<void**>(&c->refs), static_cast<size_t>(c->n_pages) * 4, 0},
      {&c->work, work_bytes(c), 0},
  };
  for (const auto& w : want) *w.p = nullptr;
  c->owned = 1;
  c->work_bytes = work_bytes(c);
  for (const auto& w : want) {
    if (pl_module::alloc(w.p, w.bytes) != cudaSuccess) {
      cudaGetLastError();
      pl_kv8_release(c);
      return PL_ENOMEM;
    }
    if (cudaMemset(*w.p, w.fill, w.bytes) != cudaSuccess) {
      pl_kv8_release(c);
      return PL_ECUDA;
    }
  }
  if (cudaDeviceSynchronize() != cudaSuccess) {
    pl_kv8_release(c);
    return PL_ECUDA;
  }
  return PL_OK;
}

void pl_kv8_release(pl_kv8* c) {
  if (!c || !c->owned) return;
  cudaFree(c->codes);
  cudaFree(c->scales);
  cudaFree(c->table);
  cudaFree(c->lens);
  cudaFree(c->refs);
  cudaFree(c->work);
  c->codes = c->work = nullptr;
  c->scales = nullptr;
  c->table = c->lens = c->refs = nullptr;
  c->work_bytes = 0;
  c->owned = 0;
}

int pl_kv8_resize_dev(const pl_kv8* c, int n, const int* d_seqs, const int* d_len, void* stream) {
  const int rc = check_kv8(c);
  if (rc) return rc;
  if (n < 0 || n > pl::kPlanSeqs || (n && !d_seqs)) return PL_EARG;
  return n ? plan(c, pl::PLAN_RESIZE, n, d_seqs, d_len, d_len != nullptr, stream) : PL_OK;
}

int pl_kv8_fork_dev(const pl_kv8* c, int n, const int* d_src, const int* d_dst, void* stream) {
  const int rc = check_kv8(c);
  if (rc) return rc;
  if (n < 0 || n > pl::kPlanSeqs || (n && (!d_src || !d_dst))) return PL_EARG;
  return n ? plan(c, pl::PLAN_FORK, n, d_src, d_dst, false, stream) : PL_OK;
}

int pl_kv8_compact_dev(const pl_kv8* c, void* stream) {
  const int rc = check_kv8(c);
  return rc ? rc : plan(c, pl::PLAN_COMPACT, 0, nullptr, nullptr, true, stream);
}

int pl_kv8_copy_dev(const pl_kv8* c, int n, const int* d_src, const int* d_dst, void* stream) {
  const int rc = check_kv8(c);
  if (rc) return rc;
  if (n < 0 || n > c->n_pages || (n && (!d_src || !d_dst))) return PL_EARG;
  return n ? plan(c, pl::PLAN_COPY, n, d_src, d_dst, true, stream) : PL_OK;
}

int pl_kv8_append_dev(const pl_kv8* c, int layer, int n, const int* d_seqs, const int* d_start,
                      int total, int max_tok, int dtype, const void* d_k, long long k_stride,
                      const void* d_v, long long v_stride, void* stream) {
  bool none = false;
  const int rc = check_call(c, layer, n, d_seqs, d_start, total, max_tok, dtype, &none);
  if (rc || none) return rc;
  if (!good_rows(d_k, k_stride, c->n_kv_heads, c->head_dim, dtype) ||
      !good_rows(d_v, v_stride, c->n_kv_heads, c->head_dim, dtype))
    return PL_EARG;
  pl::Kv8AppendArgs a;
  a.g = geo(c, layer);
  a.rope = c->rope;
  a.n = n;
  a.total = total;
  a.max_tok = max_tok;
  a.seqs = d_seqs;
  a.start = d_start;
  a.k = d_k;
  a.v = d_v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  return by_type<Append>(c, dtype, a, stream);
}

int pl_kv8_attend_dev(const pl_kv8* c, int layer, int n, const int* d_seqs, const int* d_start,
                      int total, int max_tok, int dtype, const void* d_q, long long q_stride,
                      void* d_out, long long out_stride, void* stream) {
  bool none = false;
  const int rc = check_call(c, layer, n, d_seqs, d_start, total, max_tok, dtype, &none);
  if (rc || none) return rc;
  if (!good_rows(d_q, q_stride, c->n_heads, c->head_dim, dtype) ||
      !good_rows(d_out, out_stride, c->n_heads, c->head_dim, dtype))
    return PL_EARG;
  return by_type<Attend>(c, dtype, attn_args(c, layer, n, d_seqs, d_start, total, max_tok, d_q,
                                             q_stride, d_out, out_stride), stream);
}

int pl_kv8_decode_dev(const pl_kv8* c, int layer, int n, const int* d_seqs, int dtype,
                      const void* d_q, long long q_stride, const void* d_k, long long k_stride,
                      const void* d_v, long long v_stride, void* d_out, long long out_stride,
                      void* stream) {
  bool none = false;
  const int rc = check_call(c, layer, n, d_seqs, nullptr, n, 1, dtype, &none);
  if (rc || none) return rc;
  if (!good_rows(d_q, q_stride, c->n_heads, c->head_dim, dtype) ||
      !good_rows(d_k, k_stride, c->n_kv_heads, c->head_dim, dtype) ||
      !good_rows(d_v, v_stride, c->n_kv_heads, c->head_dim, dtype) ||
      !good_rows(d_out, out_stride, c->n_heads, c->head_dim, dtype))
    return PL_EARG;
  pl::Kv8DecodeArgs d = {};
  d.a = attn_args(c, layer, n, d_seqs, nullptr, n, 1, d_q, q_stride, d_out, out_stride);
  d.k = d_k;
  d.v = d_v;
  d.k_stride = k_stride;
  d.v_stride = v_stride;
  return by_type<Decode>(c, dtype, d, stream);
}

int pl_kv8_read_dev(const pl_kv8* c, int layer, int n, const int* d_seqs, const int* d_row0,
                    const int* d_start, int total, int max_rows, int dtype, void* d_k,
                    long long k_stride, void* d_v, long long v_stride, void* stream) {
  bool none = false;
  const int rc = check_call(c, layer, n, d_seqs, d_start, total, max_rows, dtype, &none);
  if (rc || none) return rc;
  if (!d_row0 || !good_rows(d_k, k_stride, c->n_kv_heads, c->head_dim, dtype) ||
      !good_rows(d_v, v_stride, c->n_kv_heads, c->head_dim, dtype))
    return PL_EARG;
  pl::Kv8ReadArgs a;
  a.g = geo(c, layer);
  a.n = n;
  a.total = total;
  a.max_rows = max_rows;
  a.seqs = d_seqs;
  a.row0 = d_row0;
  a.start = d_start;
  a.k = d_k;
  a.v = d_v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  return by_type<Read>(c, dtype, a, stream);
}

int pl_kv8_status(const pl_kv8* c, void* stream) {
  const int rc = check_kv8(c);
  if (rc) return rc;
  // all in the stream's order: a stream that does not wait for the default
  // one could otherwise see the clearing after its next call
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t w = 0;
  uint32_t* err = &static_cast<pl::Kv8Head*>(c->work)->err;
  PL_CUDA(cudaMemcpyAsync(&w, err, sizeof(w), cudaMemcpyDeviceToHost, st));
  PL_CUDA(cudaStreamSynchronize(st));
  if (w) PL_CUDA(cudaMemsetAsync(err, 0, sizeof(w), st));
  if (w & (pl::ERR_TIMEOUT_FULL | pl::ERR_TIMEOUT_EMPTY | pl::ERR_TIMEOUT_MMA)) {
    // a block that gave up has not counted itself
    PL_CUDA(cudaMemsetAsync(work_arrived(c), 0, arrive_bytes(c), st));
    return PL_ETIMEOUT;
  }
  if (w & pl::ERR_BAD_ARG) return PL_EARG;
  if (w & pl::ERR_NO_PAGES) return PL_ENOMEM;
  return w ? PL_EFAIL : PL_OK;
}

}  // extern "C"
