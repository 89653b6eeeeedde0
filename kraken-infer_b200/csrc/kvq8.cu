// kvq8.cu -- operators over the paged 8-bit KV cache: append with rotation,
// reading pages back, and attention.  The C ABI's checks come first in each
// entry; nothing is launched for arguments outside the documented ranges.
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "kib_ctx.cuh"
#include <cudaTypedefs.h>

#include "kvq8_many.cuh"
#include "per_device.hpp"

namespace kib {
namespace {

// ------------------------------------------------------------------ append

struct Kvq8AppendParams {
  Kvq8Cache c;
  Kvq8Batch b;
  const void *q, *k, *v;
  void* q_out;
  int heads, q_parts;                                   // query heads; CTAs that share them
  int64_t q_stride, k_stride, v_stride, q_out_stride;   // elements between rows
  const float* inv_freq;                                // [pairs]
  int pairs;                                            // 0: no rotation
  int sec0, sec1, sec2, sec_total;
  const int32_t* positions;                             // [4][rows], or null: the cache position
};

// The reduction of a page's largest value: a finite |x|; NaN and infinities
// do not set a scale.
KIB_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}

// code = rint(x / s) held to [-127, 127]; NaN (an infinity over a scale of 0
// among it) gives 0.
KIB_DEV int quantise(float x, float inv) {
  const float y = __fmul_rn(x, inv);
  return y == y ? __float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f)) : 0;
}

// A CTA takes a span of positions, whole pages (64 positions, or a page of
// 128), of one sequence and one K head, one V head or kAppendQ query heads,
// for which the cosines and sines of the span are made once in shared memory.
// A row is read in 16-byte pieces by LPR lanes (a warp has 32 / LPR rows at a
// time); K and V rows stay in registers between the reduction of a page's
// largest value and the rounding, so every row is read once.  Where the rotated
// pairs lie a whole number of pieces apart, a lane gets its partners by
// shuffles.  Bound by the bytes of the rows in large calls (8192 fp32 tokens, 8
// query and 2 KV heads of 256: 36.6 us, 4.7 TB/s; queries in a launch of their
// own 14 us more), by the latency of page lookup, row, reduction and store in
// small ones (32 slots of one token: 4 us).
template <typename T, int HD>
struct AppendShape {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));    // values of a piece
  static constexpr int LPR = HD / E < 32 ? HD / E : 32;         // lanes of a row
  static constexpr int NC = HD / (E * LPR);                     // pieces of a lane
  static constexpr int RPW = 32 / LPR;                          // rows of a warp at a time
  static constexpr int ROWS = 8 / RPW;                          // times that to cover a warp's part of a page
  static constexpr int HELD = ROWS * NC * E;                    // values that a thread holds
  static constexpr int U = HELD >= 64 ? 4 : 2;                  // query rows a lane has in flight
  // small rows leave registers for four CTAs of 256 threads: such calls are bound by latency
  static constexpr int MINB = HELD >= 64 ? 1 : 2;               // of 512 threads
};
constexpr int kAppendSpan = 64;
constexpr int kAppendQ = 4;

template <int E>
KIB_DEV void store_piece_codes(int8_t* p, const int (&c)[E]) {
  uint32_t w[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i)
    w[i] = (c[4 * i] & 255) | (c[4 * i + 1] & 255) << 8 | (c[4 * i + 2] & 255) << 16 | (c[4 * i + 3] & 255) << 24;
  if constexpr (E == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

template <typename T, int HD>
__global__ void __launch_bounds__(512, AppendShape<T, HD>::MINB) kvq8_append_kernel(const __grid_constant__ Kvq8AppendParams p) {
  using Sh = AppendShape<T, HD>;
  constexpr int E = Sh::E, LPR = Sh::LPR, NC = Sh::NC, RPW = Sh::RPW, ROWS = Sh::ROWS;
  extern __shared__ __align__(16) float2 s_cs[];  // [rows of the span][pairs]
  __shared__ float s_max[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int rl = lane / LPR, cl = lane % LPR;
  const int seq = blockIdx.z, kvh = p.c.kv_heads;
  const Kvq8Seq s = kvq8_seq(p.b, seq);
  const int start = s.length - s.n, begin = max(start, 0);  // positions before 0 have no place
  const int span = max(kAppendSpan, p.c.page_tokens);
  const int base = (begin / span + static_cast<int>(blockIdx.x)) * span;
  // (a row past max_rows, the host's bound and that of s_cs, is left out)
  const int lo = max(begin, base), hi = min(min(s.length, base + span), lo + p.b.max_rows);
  if (lo >= hi) return;
  const int part = blockIdx.y;  // query heads, K heads, V heads
  const bool is_q = part < p.q_parts, is_v = part >= p.q_parts + kvh;
  const int head = part - (is_q ? 0 : p.q_parts + (is_v ? kvh : 0));
  const int half = is_v ? 0 : p.pairs;
  // rotated pairs within the first piece of each lane, a whole number of lanes apart
  const bool quick = half % E == 0 && 2 * half <= LPR * E;

  // this warp's page and rows
  const int wpp = warps * p.c.page_tokens / span, page_base = base + warp / wpp * p.c.page_tokens, wi = warp % wpp;
  auto row_pos = [&](int i) { return page_base + (i * wpp + wi) * RPW + rl; };
  const T* in = static_cast<const T*>(is_v ? p.v : p.k) + static_cast<int64_t>(head) * HD + cl * E;
  const int64_t stride = is_v ? p.v_stride : p.k_stride;
  float x[ROWS][NC][E];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int pos = row_pos(i);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][n][e] = 0.0f;
      if (!is_q && pos >= lo && pos < hi) load_vec<T, E>(in + (s.first + pos - start) * stride + n * LPR * E, x[i][n]);
    }
  }
  // the new rows of this warp's page, and its scale: all warps read it before the barrier that the writer passes
  const int first = max(lo, page_base), last = min(hi, page_base + p.c.page_tokens);
  const int page = !is_q && first < last ? kvq8_page(p.c, p.b, seq, page_base >> p.c.page_shift) : -1;
  float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + static_cast<int64_t>(max(page, 0)) * kvh + (is_q ? 0 : head);
  // a page whose first position is new is taken over: its old scale is no longer anyone's
  const float old = page >= 0 && first > page_base ? *scale : 0.0f;
  if (half) {
    // a thread keeps its pair and goes down the rows
    const int rows = static_cast<int>(blockDim.x) / half, j = static_cast<int>(threadIdx.x) % half;
    int stream = 0;
    if (p.positions && p.sec_total) {
      const int sector = j % p.sec_total;
      stream = sector < p.sec0 ? 0 : (sector < p.sec0 + p.sec1 ? 1 : (sector < p.sec0 + p.sec1 + p.sec2 ? 2 : 3));
    }
    const float freq = p.inv_freq[j];
    const int32_t* given = p.positions ? p.positions + static_cast<int64_t>(stream) * p.b.rows + s.first - start : nullptr;
    for (int r = static_cast<int>(threadIdx.x) / half; r < hi - lo && static_cast<int>(threadIdx.x) < rows * half; r += rows) {
      const int pos = given ? given[lo + r] : lo + r;
      float sn, cs;
      sincosf(__fmul_rn(static_cast<float>(pos), freq), &sn, &cs);
      s_cs[r * half + j] = make_float2(cs, sn);
    }
    __syncthreads();
  }
  // Rotates the pieces v of the row at `row` (its first value) and position
  // pos; each product is rounded by itself, as the element-wise form does.
  // Every lane of the warp takes part.
  auto rotate = [&](float (&v)[NC][E], const T* row, int pos, bool live) {
    const float2* cs = s_cs + (pos - lo) * half;
    if (quick) {
      const int d = cl * E, off = half / E;
      const bool upper = d >= half, in_pairs = d < 2 * half;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = __shfl_sync(0xffffffffu, v[0][e], in_pairs ? (upper ? lane - off : lane + off) : lane);
      if (live && in_pairs) {
        cs += upper ? d - half : d;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float4 f = *reinterpret_cast<const float4*>(cs + e);
          const float c2[2] = {f.x, f.z}, s2[2] = {f.y, f.w};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float a = __fmul_rn(v[0][e + u], c2[u]), b = __fmul_rn(o[e + u], s2[u]);
            v[0][e + u] = upper ? __fadd_rn(a, b) : __fsub_rn(a, b);
          }
        }
      }
    } else if (live) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int d = n * LPR * E + cl * E + e;
          if (d >= 2 * half) continue;
          const bool upper = d >= half;
          const float2 f = cs[upper ? d - half : d];
          const float o = to_f32<T>(row[upper ? d - half : d + half]);
          const float a = __fmul_rn(v[n][e], f.x), b = __fmul_rn(o, f.y);
          v[n][e] = upper ? __fadd_rn(a, b) : __fsub_rn(a, b);
        }
    }
  };
  if (is_q) {
    // query heads, U items (row, head) a lane in flight
    const int h0 = head * kAppendQ, share = min(kAppendQ, p.heads - h0);
    const bool in_place = p.q == p.q_out;  // then what is not rotated stays where it is
    const int items = (hi - lo) * share, step = warps * RPW;
    constexpr int U = Sh::U;
#pragma unroll 1
    for (int i0 = warp * RPW; i0 < items; i0 += U * step) {
      float y[U][NC][E];
      int row[U], pos[U], h[U];
      bool live[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int item = i0 + u * step + rl, r = item / share;
        live[u] = item < items;
        pos[u] = lo + r;
        row[u] = s.first + pos[u] - start;
        h[u] = h0 + item - r * share;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
          for (int e = 0; e < E; ++e) y[u][n][e] = 0.0f;
          const int d = n * LPR * E + cl * E;
          if (live[u] && !(in_place && d >= 2 * half))
            load_vec<T, E>(static_cast<const T*>(p.q) + row[u] * p.q_stride + static_cast<int64_t>(h[u]) * HD + d, y[u][n]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (half) rotate(y[u], static_cast<const T*>(p.q) + row[u] * p.q_stride + static_cast<int64_t>(h[u]) * HD, pos[u], live[u]);
      __syncwarp();  // in place: every lane of a row has its partners' values before the row is written
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          const int d = n * LPR * E + cl * E;
          if (live[u] && !(in_place && d >= 2 * half))
            store_vec<T, E>(static_cast<T*>(p.q_out) + row[u] * p.q_out_stride + static_cast<int64_t>(h[u]) * HD + d, y[u][n]);
        }
    }
    return;
  }
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int pos = row_pos(i);
    const bool live = pos >= lo && pos < hi;
    if (half) rotate(x[i], in - cl * E + (s.first + pos - start) * stride, pos, live);
    if (live) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) big = fmaxf(big, finite_abs(x[i][n][e]));
    }
  }
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (page >= 0) {
    for (int w = warp / wpp * wpp, i = 0; i < wpp; ++i) big = fmaxf(big, s_max[w + i]);
  }
  if (page >= 0) {
    const float now = fmaxf(old, __fmul_rn(big, 1.0f / 127.0f));
    if (wi == 0 && lane == 0) *scale = now;
    // the reciprocal of a scale below 2^-128 would be infinite: such rows and their scale are taken 2^64 times
    const bool tiny = now < 0x1p-100f;
    const float inv = now > 0.0f ? __fdiv_rn(1.0f, tiny ? now * 0x1p64f : now) : 0.0f;
    if (tiny) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int e = 0; e < E; ++e) x[i][n][e] *= 0x1p64f;
    }
    const float ratio = now > 0.0f ? __fdiv_rn(old, now) : 0.0f;
    const bool again = now != old || now == 0.0f;
    int8_t* codes = (is_v ? p.c.v : p.c.k) + page * p.c.page_stride + head * p.c.head_stride + cl * E;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int pos = row_pos(i);
      int8_t* at = codes + (pos - page_base) * p.c.token_stride;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        int c[E];
        if (pos >= first && pos < last) {
#pragma unroll
          for (int e = 0; e < E; ++e) c[e] = quantise(x[i][n][e], inv);
          store_piece_codes<E>(at + n * LPR * E, c);
        } else if (pos < first && again) {
          // codes that the page already holds move to its grown scale
          load_codes<E>(at + n * LPR * E, c);
#pragma unroll
          for (int e = 0; e < E; ++e) c[e] = __float2int_rn(__fmul_rn(static_cast<float>(c[e]), ratio));
          store_piece_codes<E>(at + n * LPR * E, c);
        }
      }
    }
  }
}

// ------------------------------------------------------------- read pages

// A thread per 16 codes; out [count][kv_heads][page_tokens][head_dim].
template <typename T, int HD>
__global__ void __launch_bounds__(256) kvq8_read_kernel(const __grid_constant__ Kvq8Cache c, const int32_t* ids, int64_t total,
                                                        T* k_out, T* v_out) {
  constexpr int CH = HD / 16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / CH;
  const int ch = static_cast<int>(i % CH), t = static_cast<int>(row & (c.page_tokens - 1));
  const int64_t ph = row >> c.page_shift;
  const int64_t at = ph / c.kv_heads;
  const int head = static_cast<int>(ph - at * c.kv_heads), page = ids[at];
  T* dst = (blockIdx.y ? v_out : k_out) + i * 16;
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  float s = 0.0f;
  if (page >= 0 && page < c.pages) {
    w = *reinterpret_cast<const uint4*>((blockIdx.y ? c.v : c.k) + page * c.page_stride + head * c.head_stride +
                                        t * c.token_stride + 16 * ch);
    s = (blockIdx.y ? c.v_scale : c.k_scale)[static_cast<int64_t>(page) * c.kv_heads + head];
  }
  const uint32_t word[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float x[8];
#pragma unroll
    // 0x4b0000bb is 2^23 + bb; bb = code + 128
    for (int e = 0; e < 8; ++e)
      x[e] = (__uint_as_float(__byte_perm(word[2 * j + e / 4], 0x4b000000u, 0x7440u + e % 4)) - 8388736.0f) * s;
    store_vec<T, 8>(dst + 8 * j, x);
  }
}

// Dynamic shared memory above 48 KB has to be asked for, once per kernel and device.
template <typename... KArgs>
cudaError_t allow_smem(int device, void (*kernel)(KArgs...), size_t bytes, PerDevice* done) {
  cudaError_t e = cudaSuccess;
  done->once(device, [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    return e == cudaSuccess;
  });
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
cudaError_t few_launch(const Kvq8AttnParams& p, const kib_ctx* ctx, cudaStream_t st) {
  static PerDevice ready;
  cudaError_t e = allow_smem(ctx->device, kvq8_few_kernel<T, HD, NT>, few_smem<T, HD, NT>(), &ready);
  if (e != cudaSuccess) return e;
  const int ctas = std::min(ctx->num_sms, kMergeMaxCtas);
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
cudaError_t few_launch_nt(const Kvq8AttnParams& p, const kib_ctx* ctx, cudaStream_t st) {
  const int nt = few_nt(p.c, p.b, p.group);
  if (nt == 1) return few_launch<T, HD, 1>(p, ctx, st);
  if constexpr (few_max_nt(HD) > 2) {
    if (nt == 3) return few_launch<T, HD, 3>(p, ctx, st);
  }
  return few_launch<T, HD, 2>(p, ctx, st);
}

// The workspace of the few-row path: records, then fp32 rows' sums.
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
size_t few_records(const Kvq8Cache& c, const Kvq8Batch& b, int group, int num_sms) {
  return up256(static_cast<size_t>(std::min(num_sms, kMergeMaxCtas)) * 2 * 8 * few_nt(c, b, group) *
               static_cast<size_t>(c.head_dim + 2) * sizeof(float));
}
size_t few_workspace(const Kvq8Cache& c, const Kvq8Batch& b, int type, int group, int num_sms) {
  const int nt = few_nt(c, b, group);
  size_t bytes = few_records(c, b, group, num_sms);
  if (type == KIB_TYPE_F32 && few_banks<float>(c.head_dim))
    bytes += static_cast<size_t>(std::min(num_sms, kMergeMaxCtas)) * few_warps_of(c.head_dim, nt) * 8 * nt * c.head_dim * sizeof(float);
  return bytes;
}

// Rows (times the group) up to which a sequence is the few-row kernel's.
constexpr int kFewLimit = 64;
// Batches with a sequence of more rows than that go to the many-row path where
// it is the faster one, reckoned in granules of 128 keys and 16 query rows per
// SM.  The few-row kernel takes the granules and about six for the start and
// end of each unit.  The many-row path takes eight for its three launches (ten
// and twelve of the shorter ones of 128 and 64 dimensions), two for 128 rows of a
// granule, and 0.2 (0.3, 0.4) for every CTA that a unit is spread over, whose
// records are joined one after another.  8 query and 2 KV heads, few against
// many, us (rows of each sequence, after its other tokens):
//                              fp32 256    fp32 64     half 256    half 64
//     1 x 100                  17   30     13   18     15   25     11   16
//     1 x 32 after 16000       54   78     28   45     42   68     22   44
//     1 x 64 after 8000        55   55     30   33     43   48     23   31
//     4 x 100                  35   34     18   21     32   28     16   19
//     4 x 64 after 1000        49   42     26   27     41   37     21   25
//     1 x 200 after 1300       51   42     28   24     41   35     21   23
//     1 x 500                  59   38     32   23     51   33     26   21
//     30 x 20 after 480        72   49     39   30     62   42     31   27
// Over 22 such batches, three head sizes and both types the rule takes 1 % more
// time than the faster kernel would (16 % at most: 150 rows after 2850, fp32 128).
bool any_many(const Kvq8Cache& c, const Kvq8Batch& b, int group, int num_sms) {
  if (static_cast<int64_t>(b.max_rows) * group <= kFewLimit || b.max_length == 0) return false;
  const int64_t rows = static_cast<int64_t>(b.rows) * group, granules = (static_cast<int64_t>(b.max_length) + kFewGranule - 1) / kFewGranule;
  const double few_units = static_cast<double>(rows / 16 + b.sequences) * c.kv_heads / num_sms;
  const double units = static_cast<double>(rows / kManyRows + b.sequences) * c.kv_heads / num_sms;
  const double spread = units < 1.0 ? std::min(1.0 / units, static_cast<double>(granules)) : 1.0;
  const double start = c.head_dim == 256 ? 8.0 : (c.head_dim == 128 ? 10.0 : 12.0), join = c.head_dim == 256 ? 0.2 : (c.head_dim == 128 ? 0.3 : 0.4);
  return few_units * static_cast<double>(granules + 6) > start + join * spread + 2.0 * units * static_cast<double>(granules);
}

// The workspace of the many-row path, in this order behind the records.
struct ManyLayout {
  size_t k16, v16, scales, seq_off, units, cum, cta_unit, split, count, bytes;
  int64_t tot_pad, max_units;
};
ManyLayout many_layout(const Kvq8Cache& c, const Kvq8Batch& b, int64_t total_length, int type, int group, int num_sms) {
  ManyLayout m = {};
  const int64_t bound = static_cast<int64_t>(b.max_length) * b.sequences;
  if (total_length <= 0 || total_length > bound) total_length = bound;
  m.tot_pad = (total_length + kManyKeys - 1) / kManyKeys * kManyKeys + static_cast<int64_t>(b.sequences) * kManyKeys;
  m.max_units = (static_cast<int64_t>(b.rows) * group / kManyRows + b.sequences) * c.kv_heads;
  const size_t codes = static_cast<size_t>(m.tot_pad) * c.kv_heads * c.head_dim * sizeof(__half);
  size_t at = up256(std::max(static_cast<size_t>(num_sms) * 2 * kManyRows * (c.head_dim + 2) * sizeof(float),
                             few_workspace(c, b, type, group, num_sms)));
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
cudaError_t many_launch(const Kvq8AttnParams& a, const ManyLayout& w, uint8_t* ws, const kib_ctx* ctx, cudaStream_t st) {
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;
  using Sh = ManyShape<HD, PL>;
  const int num_sms = ctx->num_sms;
  static PerDevice ready;
  cudaError_t e = allow_smem(ctx->device, kvq8_many_kernel<HD, PL>, Sh::kSmem, &ready);
  if (e != cudaSuccess) return e;
  if constexpr (Sh::kHeld) {
    // (a build whose launch has fewer registers would wait for the rest without end)
    static const bool enough = [] {
      cudaFuncAttributes a{};
      return cudaFuncGetAttributes(&a, kvq8_many_kernel<HD, PL>) == cudaSuccess &&
             a.numRegs * Sh::kThreads >= 128 * kManyHelperRegs + kManySoft * kManySoftRegs;
    }();
    if (!enough) return cudaErrorInvalidConfiguration;
  }
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
  p.err = ctx->d_err;
  const int kvh = a.c.kv_heads;
  CUtensorMap kmap, vmap;
  if (!tile_map(&kmap, p.k16, static_cast<int64_t>(kvh) * w.tot_pad, HD, kManyKeys) ||
      !tile_map(&vmap, p.v16, static_cast<int64_t>(kvh) * HD, w.tot_pad, HD))
    return cudaErrorInvalidValue;
  const dim3 tiles(static_cast<unsigned>(w.tot_pad / kManyKeys + 1), static_cast<unsigned>(kvh));
  kvq8_gather_kernel<HD><<<tiles, kGatherThreads, 0, st>>>(p);
  kvq8_many_kernel<HD, PL><<<num_sms, Sh::kThreads, Sh::kSmem, st>>>(kmap, vmap, p);
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

bool is_capturing(cudaStream_t st) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(st, &s) == cudaSuccess && s != cudaStreamCaptureStatusNone;
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
  // spans that max_rows consecutive positions can reach
  const int span = std::max(kAppendSpan, p.c.page_tokens);
  const unsigned spans = static_cast<unsigned>((static_cast<int64_t>(p.b.max_rows) + span - 2) / span + 1);
  p.q_parts = (p.heads + kAppendQ - 1) / kAppendQ;
  const dim3 grid(spans, static_cast<unsigned>(p.q_parts + 2 * p.c.kv_heads), static_cast<unsigned>(p.b.sequences));
  const unsigned threads = span == 128 ? 512u : 256u;
  const size_t smem = static_cast<size_t>(std::min(span, p.b.max_rows)) * p.pairs * sizeof(float2);
  cudaError_t e = cudaSuccess;
#define CALL(T, HD)                                                                                \
  do {                                                                                             \
    static PerDevice ready;                                                                        \
    e = allow_smem(ctx->device, kvq8_append_kernel<T, HD>, static_cast<size_t>(128) * (HD / 2) * sizeof(float2), &ready); \
    if (e == cudaSuccess) kvq8_append_kernel<T, HD><<<grid, threads, smem, op_stream(ctx, stream)>>>(p);   \
  } while (0)
  KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  if (e != cudaSuccess) return check_cuda(ctx, e, "kvq8_append");
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
  KIB_ARG(count < (1ull << 38) / (static_cast<uint64_t>(c.kv_heads) * c.page_tokens * (c.head_dim / 16)),
          "kvq8_read_pages: count out of range");
  const int64_t total = static_cast<int64_t>(count) * c.kv_heads * c.page_tokens * (c.head_dim / 16);
  const dim3 grid(static_cast<unsigned>((total + 255) / 256), 2);
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
  *bytes = few_workspace(c, b, type, group, ctx->num_sms);
  if (any_many(c, b, group, ctx->num_sms)) {
    const ManyLayout m = many_layout(c, b, static_cast<int64_t>(batch->total_length), type, group, ctx->num_sms);
    KIB_ARG(m.tot_pad * c.kv_heads < (1ll << 31) && m.max_units < (1ll << 27),
            "kvq8_attention: total_length or rows too large for one call");
    *bytes = m.bytes;
  }
  return KIB_OK;
}

int kib_kvq8_attention_captured(kib_ctx* ctx, const void* workspace, void* stream, int* captured, int* capturing) {
  KIB_REQUIRE_CTX(ctx);
  KIB_ARG(captured && capturing, "kvq8_attention_captured: null result");
  *captured = workspace && std::find(ctx->captured.begin(), ctx->captured.end(), workspace) != ctx->captured.end();
  *capturing = is_capturing(op_stream(ctx, stream));
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
  if (p.b.sequences == 0 || p.b.rows == 0) return KIB_OK;
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
  p.bank = reinterpret_cast<float4*>(static_cast<uint8_t*>(workspace) + few_records(p.c, p.b, p.group, ctx->num_sms));
  p.err = ctx->d_err;
  const cudaStream_t st = op_stream(ctx, stream);
  // a graph will replay on this workspace
  if (is_capturing(st) && workspace && std::find(ctx->captured.begin(), ctx->captured.end(), workspace) == ctx->captured.end())
    ctx->captured.push_back(workspace);
  const bool many = any_many(p.c, p.b, p.group, ctx->num_sms);
  // one sequence of many rows needs one path; a mixed batch takes both, each its own sequences
  p.few_limit = many ? (p.b.sequences == 1 ? 0 : kFewLimit) : 0x7fffffff;
  cudaError_t e = cudaSuccess;
  if (p.few_limit > 0) {
#define CALL(T, HD) e = few_launch_nt<T, HD>(p, ctx, st)
    KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  }
  if (many && e == cudaSuccess) {
    const ManyLayout m = many_layout(p.c, p.b, static_cast<int64_t>(batch->total_length), type, p.group, ctx->num_sms);
#define CALL(T, HD) e = many_launch<T, HD>(p, m, static_cast<uint8_t*>(workspace), ctx, st)
    KVQ8_DISPATCH(type, p.c.head_dim, CALL);
#undef CALL
  }
  if (e != cudaSuccess) return check_cuda(ctx, e, "kvq8_attention");
  return finish(ctx, stream, "kvq8_attention");
}

}  // extern "C"
