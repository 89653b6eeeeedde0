// kvq8.cu -- operators over the paged 8-bit KV cache: append with rotation,
// reading pages back, and attention.  The C ABI's checks come first in each
// entry; nothing is launched for arguments outside the documented ranges.
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "kib_ctx.cuh"
#include <cudaTypedefs.h>

#include "kvq8_many.cuh"

namespace kib {
namespace {

// ------------------------------------------------------------------ append

struct Kvq8AppendParams {
  Kvq8Cache c;
  Kvq8Batch b;
  const void *q, *k, *v;
  void* q_out;
  int heads;
  int64_t q_stride, k_stride, v_stride, q_out_stride;  // elements between rows
  const float* inv_freq;  // [pairs]
  int pairs;              // 0: no rotation
  int sec0, sec1, sec2, sec_total;
  const int32_t* positions;  // [4][rows], or null: the cache position
};

// The reduction of a page's largest value: a finite |x|; NaN and infinities
// do not set a scale.
KIB_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}

// code = rint(x / s) held to [-127, 127]; NaN gives 0.
KIB_DEV int quantise(float x, float inv) {
  const float y = fminf(fmaxf(__fmul_rn(x, inv), -127.0f), 127.0f);
  return x == x ? __float2int_rn(y) : 0;
}

constexpr int kAppendRows = 8;      // rows of a page per warp, held in registers between the two steps
constexpr int kAppendMaxPairs = 128;

// One CTA per (run, head, sequence): a run is the new rows of one page.
// blockIdx.y counts K heads, then V heads, then query heads.  A warp holds
// whole rows (head_dim / 32 values a lane), kAppendRows of them, so rows are
// read once: the page's largest value is reduced over the CTA, then the same
// registers are rounded and stored.  Bound by the bytes of the rows.
template <typename T, int HD>
__global__ void kvq8_append_kernel(const __grid_constant__ Kvq8AppendParams p) {
  constexpr int V = HD / 32;
  __shared__ float s_max[16];
  __shared__ float2 s_cs[16][kAppendMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int seq = blockIdx.z, kvh = p.c.kv_heads;
  const Kvq8Seq s = kvq8_seq(p.b, seq);
  const int start = s.length - s.n;  // position of the sequence's first new row
  const int begin = max(start, 0);
  const int page_index = (begin >> p.c.page_shift) + static_cast<int>(blockIdx.x);
  const int base = page_index << p.c.page_shift;
  const int lo = max(begin, base), hi = min(s.length, base + p.c.page_tokens);
  if (lo >= hi) return;
  int head = blockIdx.y;
  const int what = head < kvh ? 0 : (head < 2 * kvh ? 1 : 2);  // K, V, Q
  head -= what * kvh;
  const bool rotated = p.pairs > 0 && what != 1;
  const T* in;
  int64_t stride;
  if (what == 0) in = static_cast<const T*>(p.k), stride = p.k_stride;
  else if (what == 1) in = static_cast<const T*>(p.v), stride = p.v_stride;
  else in = static_cast<const T*>(p.q), stride = p.q_stride;
  in += static_cast<int64_t>(head) * HD;

  float x[kAppendRows][V];
  const int r0 = lo - base + ((warp - (lo - base)) % warps + warps) % warps;  // this warp's rows: r0, r0 + warps, ..
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int r = r0 + i * warps;
    if (base + r < hi) load_vec<T, V>(in + (s.first + base + r - start) * stride + lane * V, x[i]);
  }
  if (rotated) {
    const int half = p.pairs, e0 = lane * V;
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
      const int r = r0 + i * warps;
      if (base + r >= hi) continue;
      const int row = s.first + base + r - start;
      for (int j = lane; j < half; j += 32) {
        int pos = base + r;
        if (p.positions) {
          const int sector = p.sec_total ? j % p.sec_total : 0;
          const int stream = sector < p.sec0 ? 0 : (sector < p.sec0 + p.sec1 ? 1 : (sector < p.sec0 + p.sec1 + p.sec2 ? 2 : 3));
          pos = p.positions[static_cast<int64_t>(p.sec_total ? stream : 0) * p.b.rows + row];
        }
        float sn, cs;
        sincosf(__fmul_rn(static_cast<float>(pos), p.inv_freq[j]), &sn, &cs);
        s_cs[warp][j] = make_float2(cs, sn);
      }
      __syncwarp();
      const T* xr = in + static_cast<int64_t>(row) * stride;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int d = e0 + e;
        if (d < 2 * half) {
          const bool upper = d >= half;
          const float2 cs = s_cs[warp][upper ? d - half : d];
          const float o = to_f32<T>(xr[upper ? d - half : d + half]);
          // each product rounded by itself, as the element-wise form does
          x[i][e] = upper ? __fadd_rn(__fmul_rn(x[i][e], cs.x), __fmul_rn(o, cs.y))
                          : __fsub_rn(__fmul_rn(x[i][e], cs.x), __fmul_rn(o, cs.y));
        }
      }
      __syncwarp();
    }
  }
  if (what == 2) {
    T* out = static_cast<T*>(p.q_out) + static_cast<int64_t>(head) * HD;
    // q_out may be q itself: every lane of a row has read its partner's value
    // before the row is written (the warp is in step after the rotation)
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
      const int r = r0 + i * warps;
      if (base + r < hi) store_vec<T, V>(out + (s.first + base + r - start) * p.q_out_stride + lane * V, x[i]);
    }
    return;
  }
  const int page = kvq8_page(p.c, p.b, seq, page_index);
  if (page < 0) return;
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    if (base + r0 + i * warps < hi) {
#pragma unroll
      for (int e = 0; e < V; ++e) big = fmaxf(big, finite_abs(x[i][e]));
    }
  }
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  float* scale = (what == 0 ? p.c.k_scale : p.c.v_scale) + static_cast<int64_t>(page) * kvh + head;
  // a run that begins at the page's first row takes the page over: its old scale is no longer anyone's
  const float old = lo > base ? *scale : 0.0f;
  __syncthreads();
  big = s_max[0];
  for (int w = 1; w < warps; ++w) big = fmaxf(big, s_max[w]);
  const float now = fmaxf(old, __fmul_rn(big, 1.0f / 127.0f));
  if (threadIdx.x == 0) *scale = now;
  const float inv = now > 0.0f ? __fdiv_rn(1.0f, now) : 0.0f;
  int8_t* codes = (what == 0 ? p.c.k : p.c.v) + page * p.c.page_stride + head * p.c.head_stride + lane * V;
  if (now != old || now == 0.0f) {
    const float ratio = now > 0.0f ? __fdiv_rn(old, now) : 0.0f;
    for (int r = warp; r < lo - base; r += warps) {
      int c[V];
      load_codes<V>(codes + r * p.c.token_stride, c);
#pragma unroll
      for (int e = 0; e < V; ++e) c[e] = __float2int_rn(__fmul_rn(static_cast<float>(c[e]), ratio));
      store_codes<V>(codes + r * p.c.token_stride, c);
    }
  }
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int r = r0 + i * warps;
    if (base + r < hi) {
      int c[V];
#pragma unroll
      for (int e = 0; e < V; ++e) c[e] = quantise(x[i][e], inv);
      store_codes<V>(codes + r * p.c.token_stride, c);
    }
  }
}

// ------------------------------------------------------------- read pages

// One warp per row of a page and head; out [count][kv_heads][page_tokens][head_dim].
template <typename T, int HD>
__global__ void kvq8_read_kernel(const __grid_constant__ Kvq8Cache c, const int32_t* ids, int64_t total, T* k_out,
                                 T* v_out) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= total) return;
  const int t = static_cast<int>(row & (c.page_tokens - 1));
  const int64_t ph = row >> c.page_shift;
  const int head = static_cast<int>(ph % c.kv_heads), page = ids[ph / c.kv_heads];
  const bool ok = page >= 0 && page < c.pages;
  const int8_t* src = blockIdx.y ? c.v : c.k;
  T* dst = (blockIdx.y ? v_out : k_out) + row * HD + lane * V;
  float x[V] = {};
  if (ok) {
    int code[V];
    load_codes<V>(src + page * c.page_stride + head * c.head_stride + t * c.token_stride + lane * V, code);
    const float s = (blockIdx.y ? c.v_scale : c.k_scale)[static_cast<int64_t>(page) * c.kv_heads + head];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = static_cast<float>(code[e]) * s;
  }
  store_vec<T, V>(dst, x);
}

// --------------------------------------------------------------- attention

// Dynamic shared memory above 48 KB has to be asked for, once per kernel.
template <typename... KArgs>
cudaError_t allow_smem(void (*kernel)(KArgs...), size_t bytes, bool* done) {
  if (*done) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  *done = e == cudaSuccess;
  return e;
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return enc;
}

// [rows][cols] halves in boxes of box_rows x 64, 128-byte swizzle.
bool tile_map(CUtensorMap* map, const __half* base, int64_t rows, int64_t cols, int box_rows) {
  const auto enc = map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The cache's codes [page][head][token][d] in boxes of 16 tokens x 128 (64)
// dimensions, swizzled by the box's width.
bool codes_map(CUtensorMap* map, const int8_t* base, const Kvq8Cache& c) {
  const auto enc = map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_tokens),
                              static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.pages)};
  // a stride over one element is never taken, but has to be a legal one
  auto stride = [](int64_t s, bool one) { return static_cast<cuuint64_t>(one && s == 0 ? 16 : s); };
  const cuuint64_t strides[3] = {stride(c.token_stride, false), stride(c.head_stride, c.kv_heads == 1),
                                 stride(c.page_stride, c.pages == 1)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(std::min(c.head_dim, 128)), 16, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, c.head_dim >= 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, int NT>
cudaError_t few_launch(const Kvq8AttnParams& p, int num_sms, cudaStream_t st) {
  static bool ready = false;
  cudaError_t e = allow_smem(kvq8_few_kernel<T, HD, NT>, few_smem<T, HD, NT>(), &ready);
  if (e != cudaSuccess) return e;
  const int ctas = std::min(num_sms, kMergeMaxCtas);
  CUtensorMap kmap, vmap;
  if (!codes_map(&kmap, p.c.k, p.c) || !codes_map(&vmap, p.c.v, p.c)) return cudaErrorInvalidValue;
  kvq8_few_kernel<T, HD, NT><<<ctas, few_warps<HD, NT>() * 32, few_smem<T, HD, NT>(), st>>>(kmap, vmap, p);
  const int64_t rows = std::min<int64_t>(static_cast<int64_t>(p.b.max_rows) * p.group, p.few_limit);
  const int groups = static_cast<int>((rows + 8 * NT - 1) / (8 * NT));
  const dim3 grid(static_cast<unsigned>(p.b.sequences) * p.c.kv_heads * groups, static_cast<unsigned>(std::min<int64_t>(rows, 8 * NT)));
  return launch_pdl(kvq8_merge_kernel<T, HD, NT>, grid, dim3(HD), 0, st, p, ctas, groups);
}

// Eighths of a unit's rows: the fewest that hold all of a sequence's rows, as
// the cache is read once per unit; the most there are beyond that.
int few_nt(const Kvq8Cache& c, const Kvq8Batch& b, int group) {
  return static_cast<int>(std::min<int64_t>((static_cast<int64_t>(b.max_rows) * group + 7) / 8, few_max_nt(c.head_dim)));
}
template <typename T, int HD>
cudaError_t few_launch_nt(const Kvq8AttnParams& p, int num_sms, cudaStream_t st) {
  const int nt = few_nt(p.c, p.b, p.group);
  if (nt == 1) return few_launch<T, HD, 1>(p, num_sms, st);
  if constexpr (few_max_nt(HD) > 2) {
    if (nt == 3) return few_launch<T, HD, 3>(p, num_sms, st);
  }
  return few_launch<T, HD, 2>(p, num_sms, st);
}

size_t few_workspace(const Kvq8Cache& c, const Kvq8Batch& b, int group, int num_sms) {
  return static_cast<size_t>(std::min(num_sms, kMergeMaxCtas)) * 2 * 8 * few_nt(c, b, group) *
         static_cast<size_t>(c.head_dim + 2) * sizeof(float);
}

// Rows (times the group) up to which a sequence is the few-row kernel's.
constexpr int kFewLimit = 64;
bool any_many(const Kvq8Batch& b, int group) { return static_cast<int64_t>(b.max_rows) * group > kFewLimit; }

// The workspace of the many-row path, in this order behind the records.
struct ManyLayout {
  size_t k16, v16, scales, seq_off, units, cum, cta_unit, split, count, bytes;
  int64_t tot_pad, max_units;
};
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
ManyLayout many_layout(const Kvq8Cache& c, const Kvq8Batch& b, int64_t total_length, int group, int num_sms) {
  ManyLayout m = {};
  const int64_t bound = static_cast<int64_t>(b.max_length) * b.sequences;
  if (total_length <= 0 || total_length > bound) total_length = bound;
  m.tot_pad = (total_length + kManyKeys - 1) / kManyKeys * kManyKeys + static_cast<int64_t>(b.sequences) * kManyKeys;
  m.max_units = (static_cast<int64_t>(b.rows) * group / kManyRows + b.sequences) * c.kv_heads;
  const size_t codes = static_cast<size_t>(m.tot_pad) * c.kv_heads * c.head_dim * sizeof(__half);
  size_t at = up256(std::max(static_cast<size_t>(num_sms) * 2 * kManyRows * (c.head_dim + 2) * sizeof(float),
                             few_workspace(c, b, group, num_sms)));
  m.k16 = at, at = up256(at + codes);
  m.v16 = at, at = up256(at + codes);
  // one tile more: a unit without keys still reads the scales of one granule
  m.scales = at, at = up256(at + (static_cast<size_t>(m.tot_pad) * c.kv_heads + kManyKeys) / 16 * sizeof(float2));
  m.seq_off = at, at = up256(at + (static_cast<size_t>(b.sequences) + 1) * sizeof(int));
  m.units = at, at = up256(at + static_cast<size_t>(m.max_units) * sizeof(int4));
  m.cum = at, at = up256(at + (static_cast<size_t>(m.max_units) + 1) * sizeof(int64_t));
  m.cta_unit = at, at = up256(at + static_cast<size_t>(num_sms) * sizeof(int));
  m.split = at, at = up256(at + static_cast<size_t>(num_sms) * sizeof(int4));
  m.count = at, at = up256(at + 2 * sizeof(int));
  m.bytes = at;
  return m;
}

template <typename T, int HD>
cudaError_t many_launch(const Kvq8AttnParams& a, const ManyLayout& w, uint8_t* ws, int num_sms, int* err, cudaStream_t st) {
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;
  using Sh = ManyShape<HD, PL>;
  static bool ready = false;
  cudaError_t e = allow_smem(kvq8_many_kernel<HD, PL>, Sh::kSmem, &ready);
  if (e != cudaSuccess) return e;
  Kvq8ManyParams p;
  p.a = a;
  p.a.partial = reinterpret_cast<float*>(ws);
  p.tot_pad = static_cast<int>(w.tot_pad);
  p.max_units = static_cast<int>(w.max_units);
  p.k16 = reinterpret_cast<__half*>(ws + w.k16);
  p.v16 = reinterpret_cast<__half*>(ws + w.v16);
  p.scales = reinterpret_cast<float2*>(ws + w.scales);
  p.seq_off = reinterpret_cast<int*>(ws + w.seq_off);
  p.units = reinterpret_cast<int4*>(ws + w.units);
  p.cum = reinterpret_cast<int64_t*>(ws + w.cum);
  p.cta_unit = reinterpret_cast<int*>(ws + w.cta_unit);
  p.split = reinterpret_cast<int4*>(ws + w.split);
  p.count = reinterpret_cast<int*>(ws + w.count);
  p.ctas = num_sms;
  p.err = err;
  const int kvh = a.c.kv_heads;
  CUtensorMap kmap, vmap;
  if (!tile_map(&kmap, p.k16, static_cast<int64_t>(kvh) * w.tot_pad, HD, kManyKeys) ||
      !tile_map(&vmap, p.v16, static_cast<int64_t>(kvh) * HD, w.tot_pad, HD))
    return cudaErrorInvalidValue;
  const dim3 tiles(static_cast<unsigned>(w.tot_pad / kManyKeys + 1), static_cast<unsigned>(kvh));
  kvq8_gather_kernel<HD><<<tiles, kGatherThreads, 0, st>>>(p);
  kvq8_many_kernel<HD, PL><<<num_sms, kManyThreads, Sh::kSmem, st>>>(kmap, vmap, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_pdl(kvq8_many_merge<HD, PL>, dim3(static_cast<unsigned>(num_sms), kManyRows / 8), dim3(256), 0, st, p);
}

// -------------------------------------------------------------- host side

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int make_cache(kib_ctx* ctx, const kib_kvq8_cache* in, Kvq8Cache* c) {
  KIB_ARG(in, "kvq8: null cache");
  KIB_ARG(in->k && in->v && in->k_scale && in->v_scale, "kvq8: null cache pointer");
  KIB_ARG(in->head_dim == 64 || in->head_dim == 128 || in->head_dim == 256, "kvq8: head_dim must be 64, 128 or 256");
  KIB_ARG(in->page_tokens == 16 || in->page_tokens == 32 || in->page_tokens == 64 || in->page_tokens == 128,
          "kvq8: page_tokens must be 16, 32, 64 or 128");
  KIB_ARG(in->kv_heads > 0 && in->kv_heads <= 256, "kvq8: kv_heads must be in 1..256");
  KIB_ARG(in->pages > 0 && in->pages < (1ull << 31), "kvq8: pages out of range");
  c->k = in->k;
  c->v = in->v;
  c->k_scale = in->k_scale;
  c->v_scale = in->v_scale;
  c->pages = static_cast<int>(in->pages);
  c->kv_heads = static_cast<int>(in->kv_heads);
  c->page_tokens = static_cast<int>(in->page_tokens);
  c->page_shift = in->page_tokens == 16 ? 4 : in->page_tokens == 32 ? 5 : in->page_tokens == 64 ? 6 : 7;
  c->head_dim = static_cast<int>(in->head_dim);
  if (in->page_stride == 0 && in->head_stride == 0 && in->token_stride == 0) {
    c->token_stride = c->head_dim;
    c->head_stride = c->token_stride * c->page_tokens;
    c->page_stride = c->head_stride * c->kv_heads;
  } else {
    KIB_ARG(in->page_stride < (1ull << 40) && in->head_stride < (1ull << 40) && in->token_stride < (1ull << 40),
            "kvq8: cache strides out of range");
    c->page_stride = static_cast<int64_t>(in->page_stride);
    c->head_stride = static_cast<int64_t>(in->head_stride);
    c->token_stride = static_cast<int64_t>(in->token_stride);
    KIB_ARG(c->token_stride >= c->head_dim && (c->kv_heads == 1 || c->head_stride >= c->head_dim) &&
                (c->pages == 1 || c->page_stride >= c->head_dim),
            "kvq8: cache strides smaller than a row");
  }
  KIB_ARG(c->page_stride % 16 == 0 && c->head_stride % 16 == 0 && c->token_stride % 16 == 0 && aligned(in->k, 16) &&
              aligned(in->v, 16),
          "kvq8: cache pointers and strides must be multiples of 16 bytes");
  return KIB_OK;
}

int make_batch(kib_ctx* ctx, const kib_kvq8_batch* in, const Kvq8Cache& c, Kvq8Batch* b) {
  KIB_ARG(in, "kvq8: null batch");
  KIB_ARG(in->sequences <= kFewMaxSeqs && in->rows < (1ull << 31) && in->table_stride < (1ull << 31),
          "kvq8: batch dimensions out of range (at most 4096 sequences)");
  KIB_ARG(in->max_rows <= in->rows, "kvq8: max_rows exceeds rows");
  KIB_ARG(in->rows == 0 || in->max_rows > 0, "kvq8: max_rows must be positive");
  KIB_ARG(in->sequences == 0 || (in->lengths && in->row_start), "kvq8: null batch pointer");
  KIB_ARG(in->sequences == 0 || in->table_stride == 0 || in->block_table, "kvq8: null block table");
  const uint64_t most = in->table_stride * static_cast<uint64_t>(c.page_tokens);
  KIB_ARG(most < (1ull << 31), "kvq8: the block table spans more than 2^31 positions");
  b->table = in->block_table;
  b->lengths = in->lengths;
  b->row_start = in->row_start;
  b->sequences = static_cast<int>(in->sequences);
  b->table_stride = static_cast<int>(in->table_stride);
  b->rows = static_cast<int>(in->rows);
  b->max_rows = static_cast<int>(in->max_rows);
  b->max_length = static_cast<int>(in->max_length && in->max_length < most ? in->max_length : most);
  return KIB_OK;
}

// 0: packed.  Rows are read and written in 16-byte pieces.
int row_stride(kib_ctx* ctx, const void* p, uint64_t given, uint64_t packed, size_t elem, int64_t* out) {
  KIB_ARG(given == 0 || given >= packed, "kvq8: row stride smaller than a row");
  const uint64_t st = given ? given : packed;
  KIB_ARG(st < (1ull << 40) && st * elem % 16 == 0 && aligned(p, 16),
          "kvq8: row pointers and strides must be multiples of 16 bytes");
  *out = static_cast<int64_t>(st);
  return KIB_OK;
}

size_t elem_size(int type) { return type == KIB_TYPE_F32 ? 4 : type == KIB_TYPE_F16 ? 2 : 0; }

// The call's stream; on the context's own stream the call waits, like every op.
cudaStream_t op_stream(kib_ctx* ctx, void* stream) { return stream ? static_cast<cudaStream_t>(stream) : ctx->stream; }
int finish(kib_ctx* ctx, void* stream, const char* what) {
  if (!stream) return finish_op(ctx, what);
  return check_cuda(ctx, cudaGetLastError(), what);
}

#define KIB_TRY(expr)          \
  do {                         \
    const int st_ = (expr);    \
    if (st_ != KIB_OK) return st_; \
  } while (0)

// kernel<T, HD> by type and head size
#define KVQ8_DISPATCH(type, hd, CALL)                \
  do {                                               \
    if ((type) == KIB_TYPE_F32) {                    \
      if ((hd) == 64) CALL(float, 64);               \
      else if ((hd) == 128) CALL(float, 128);        \
      else CALL(float, 256);                         \
    } else {                                         \
      if ((hd) == 64) CALL(__half, 64);              \
      else if ((hd) == 128) CALL(__half, 128);       \
      else CALL(__half, 256);                        \
    }                                                \
  } while (0)

}  // namespace
}  // namespace kib

using namespace kib;

extern "C" {

int kib_kvq8_append(kib_ctx* ctx, const kib_kvq8_cache* cache, const kib_kvq8_batch* batch, const kib_rope* rope,
                    int type, uint64_t heads, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride,
                    const void* v, uint64_t v_stride, void* q_out, uint64_t q_out_stride, void* stream) {
  KIB_REQUIRE_CTX(ctx);
  Kvq8AppendParams p = {};
  KIB_TRY(make_cache(ctx, cache, &p.c));
  KIB_TRY(make_batch(ctx, batch, p.c, &p.b));
  const size_t es = elem_size(type);
  KIB_ARG(es, "kvq8_append: type must be F32(0) or F16(1)");
  if (p.b.sequences == 0 || p.b.rows == 0) return KIB_OK;
  KIB_ARG(k && v, "kvq8_append: null rows");
  KIB_ARG(!q == !q_out, "kvq8_append: q and q_out go together");
  KIB_ARG(!q || (heads > 0 && heads <= 4096), "kvq8_append: heads must be in 1..4096");
  const uint64_t hd = static_cast<uint64_t>(p.c.head_dim), kvd = hd * static_cast<uint64_t>(p.c.kv_heads);
  KIB_TRY(row_stride(ctx, k, k_stride, kvd, es, &p.k_stride));
  KIB_TRY(row_stride(ctx, v, v_stride, kvd, es, &p.v_stride));
  if (q) {
    KIB_TRY(row_stride(ctx, q, q_stride, heads * hd, es, &p.q_stride));
    KIB_TRY(row_stride(ctx, q_out, q_out_stride, heads * hd, es, &p.q_out_stride));
    KIB_ARG(q != q_out || p.q_stride == p.q_out_stride, "kvq8_append: in-place q needs one stride");
  }
  if (rope) {
    KIB_ARG(rope->pairs == 0 || rope->inv_freq, "kvq8_append: null inv_freq");
    KIB_ARG(2 * rope->pairs <= hd, "kvq8_append: more rotation pairs than half a head");
    for (uint64_t x : rope->sections) KIB_ARG(x <= hd, "kvq8_append: rotation sections out of range");
    p.inv_freq = rope->inv_freq;
    p.pairs = static_cast<int>(rope->pairs);
    p.sec0 = static_cast<int>(rope->sections[0]);
    p.sec1 = static_cast<int>(rope->sections[1]);
    p.sec2 = static_cast<int>(rope->sections[2]);
    p.sec_total = p.sec0 + p.sec1 + p.sec2 + static_cast<int>(rope->sections[3]);
    p.positions = rope->positions;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.heads = q ? static_cast<int>(heads) : 0;
  // pages that max_rows consecutive positions can reach
  const unsigned runs = static_cast<unsigned>((p.b.max_rows - 1 + p.c.page_tokens - 1) / p.c.page_tokens + 1);
  const dim3 grid(runs, static_cast<unsigned>(2 * p.c.kv_heads + p.heads), static_cast<unsigned>(p.b.sequences));
  const unsigned threads = static_cast<unsigned>(p.c.page_tokens / kAppendRows * 32);
#define CALL(T, HD) kvq8_append_kernel<T, HD><<<grid, threads, 0, op_stream(ctx, stream)>>>(p)
  KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  return finish(ctx, stream, "kvq8_append");
}

int kib_kvq8_read_pages(kib_ctx* ctx, const kib_kvq8_cache* cache, const int32_t* page_ids, uint64_t count, int type,
                        void* k_out, void* v_out, void* stream) {
  KIB_REQUIRE_CTX(ctx);
  Kvq8Cache c;
  KIB_TRY(make_cache(ctx, cache, &c));
  KIB_ARG(elem_size(type), "kvq8_read_pages: type must be F32(0) or F16(1)");
  if (count == 0) return KIB_OK;
  KIB_ARG(page_ids && k_out && v_out, "kvq8_read_pages: null pointer");
  KIB_ARG(aligned(k_out, 16) && aligned(v_out, 16), "kvq8_read_pages: outputs must be 16-byte aligned");
  KIB_ARG(count < (1ull << 31) / (static_cast<uint64_t>(c.kv_heads) * c.page_tokens / 8),
          "kvq8_read_pages: count out of range");
  const int64_t total = static_cast<int64_t>(count) * c.kv_heads * c.page_tokens;
  const dim3 grid(static_cast<unsigned>((total + 7) / 8), 2);
#define CALL(T, HD)                                                                                  \
  kvq8_read_kernel<T, HD><<<grid, 256, 0, op_stream(ctx, stream)>>>(c, page_ids, total, static_cast<T*>(k_out), \
                                                                    static_cast<T*>(v_out))
  KVQ8_DISPATCH(type, c.head_dim, CALL);
#undef CALL
  return finish(ctx, stream, "kvq8_read_pages");
}

int kib_kvq8_attention_workspace(kib_ctx* ctx, const kib_kvq8_cache* cache, const kib_kvq8_batch* batch, int type,
                                 uint64_t heads, uint64_t* bytes) {
  KIB_REQUIRE_CTX(ctx);
  Kvq8Cache c;
  Kvq8Batch b;
  KIB_TRY(make_cache(ctx, cache, &c));
  KIB_TRY(make_batch(ctx, batch, c, &b));
  KIB_ARG(bytes, "kvq8_attention_workspace: null result");
  KIB_ARG(elem_size(type), "kvq8_attention: type must be F32(0) or F16(1)");
  KIB_ARG(heads > 0 && heads <= 4096 && heads % static_cast<uint64_t>(c.kv_heads) == 0,
          "kvq8_attention: heads must be a multiple of kv_heads, at most 4096");
  KIB_ARG(static_cast<uint64_t>(b.rows) * heads < (1ull << 31), "kvq8_attention: rows times heads out of range");
  const int group = static_cast<int>(heads) / c.kv_heads;
  *bytes = few_workspace(c, b, group, ctx->num_sms);
  if (any_many(b, group)) {
    const ManyLayout m = many_layout(c, b, static_cast<int64_t>(batch->total_length), group, ctx->num_sms);
    KIB_ARG(m.tot_pad * c.kv_heads < (1ll << 31) && m.max_units < (1ll << 27),
            "kvq8_attention: total_length or rows too large for one call");
    *bytes = m.bytes;
  }
  return KIB_OK;
}

int kib_kvq8_attention(kib_ctx* ctx, const kib_kvq8_cache* cache, const kib_kvq8_batch* batch, int type,
                       uint64_t heads, const void* q, uint64_t q_stride, float scale, void* out, uint64_t out_stride,
                       void* workspace, uint64_t workspace_bytes, void* stream) {
  uint64_t need = 0;
  KIB_TRY(kib_kvq8_attention_workspace(ctx, cache, batch, type, heads, &need));
  Kvq8AttnParams p = {};
  KIB_TRY(make_cache(ctx, cache, &p.c));
  KIB_TRY(make_batch(ctx, batch, p.c, &p.b));
  if (p.b.rows == 0) return KIB_OK;
  KIB_ARG(q && out, "kvq8_attention: null rows");
  KIB_ARG(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 256))),
          "kvq8_attention: workspace too small or not 256-byte aligned");
  KIB_ARG(scale == scale && scale - scale == 0.0f, "kvq8_attention: scale is not finite");
  const size_t es = elem_size(type);
  const uint64_t row = heads * static_cast<uint64_t>(p.c.head_dim);
  KIB_TRY(row_stride(ctx, q, q_stride, row, es, &p.q_stride));
  KIB_TRY(row_stride(ctx, out, out_stride, row, es, &p.out_stride));
  p.q = q;
  p.out = out;
  p.heads = static_cast<int>(heads);
  p.group = p.heads / p.c.kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.partial = static_cast<float*>(workspace);
  p.err = ctx->d_err;
  const cudaStream_t st = op_stream(ctx, stream);
  const bool many = any_many(p.b, p.group);
  // one sequence of many rows needs one path; a mixed batch takes both, each its own sequences
  p.few_limit = many ? (p.b.sequences == 1 ? 0 : kFewLimit) : 0x7fffffff;
  cudaError_t e = cudaSuccess;
  if (p.few_limit > 0) {
#define CALL(T, HD) e = few_launch_nt<T, HD>(p, ctx->num_sms, st)
    KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  }
  if (many && e == cudaSuccess) {
    const ManyLayout m = many_layout(p.c, p.b, static_cast<int64_t>(batch->total_length), p.group, ctx->num_sms);
#define CALL(T, HD) e = many_launch<T, HD>(p, m, static_cast<uint8_t*>(workspace), ctx->num_sms, ctx->d_err, st)
    KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  }
  if (e != cudaSuccess) return check_cuda(ctx, e, "kvq8_attention");
  return finish(ctx, stream, "kvq8_attention");
}

}  // extern "C"
