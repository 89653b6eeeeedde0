// kvq8_few.cuh -- attention of few rows per sequence (single decoded tokens,
// speculative verify) over the paged 8-bit cache.
//
// For a unit (sequence, KV head, group of up to 8 NT query rows) the cache's
// codes pass once through registers:
//   S^T = K Q^T, s = S * k_scale * scale, running maximum m, p = 2^(s - m),
//   O^T += V^T (p * v_scale)^T, l += p;   out = O / l.
// Codes are integers below 128 in magnitude, exact in half, so only q and p
// are rounded: half rows use q as given and p as one half; fp32 rows use both
// as high + low halves (22 bits).  v_scale goes into p, relative to the
// largest power of two met so far (exact to move) and 2^14 above it, so p
// keeps its relative accuracy down to 2^-28 of the largest in half.
//
// Work is cut into granules of 128 keys, laid end to end over all units; each
// of the grid's CTAs takes an equal run of them, whatever the lengths are, so
// the kernel needs no host knowledge of the lengths.  A unit that crosses
// CTAs leaves partial (m, l, O) records, which kvq8_merge_kernel joins in
// order: the result depends on no timing.  Within a CTA, eight warps take
// 16-key tiles in turn, each with its own m, l and O, and join in shared
// memory at the end of the unit's run.
//
// Bound by HBM: 2 bytes per key, head and dimension.  K rows are loaded so
// that a lane's 16 bytes are the A fragments of four mma k-steps (the
// dimensions of a dot product may be taken in any order, and q is laid out
// the same way); V rows so that two byte permutes transpose 4 keys x 2
// dimensions into a fragment.  No shared memory and no barrier between the
// loads and the tensor cores: a warp has the next K rows in flight while it
// works on V, and V rows while it works on K.
#pragma once

#include "kvq8.cuh"

namespace kib {

constexpr int kFewGranule = 128;
constexpr int kFewWarps = 8;
constexpr int kFewMaxSeqs = 4096;

struct Kvq8AttnParams {
  Kvq8Cache c;
  Kvq8Batch b;
  const void* q;
  void* out;
  int heads, group;  // group = heads / kv_heads
  int64_t q_stride, out_stride;
  float scale_log2;  // softmax scale times log2(e)
  float* partial;    // [ctas][2][rows of a unit][head_dim + 2]
  int few_limit;     // sequences of at most this many rows * group are this kernel's
};

KIB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
KIB_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
KIB_DEV void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
KIB_DEV uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Bytes 0,1 (sel 0x4140) or 2,3 (0x4342) of biased codes (code + 128) as two
// halves: 0x64bb is 1024 + bb, from which 1152 leaves the code, exactly.
KIB_DEV uint32_t codes_to_half2(uint32_t biased, uint32_t sel) {
  const uint32_t h = prmt(biased, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
KIB_DEV uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
KIB_DEV uint4 ldg_stream(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Granules of one unit of a sequence, and its units per KV head.
struct FewSeq {
  int granules, groups;
};
template <int NT>
KIB_DEV FewSeq few_seq(const Kvq8AttnParams& p, int s) {
  const Kvq8Seq q = kvq8_seq(p.b, s);
  const int64_t rows = static_cast<int64_t>(q.n) * p.group;
  FewSeq f{0, 0};
  if (q.n > 0 && rows <= p.few_limit) {
    f.groups = static_cast<int>((rows + 8 * NT - 1) / (8 * NT));
    f.granules = max(1, (min(q.length, p.b.max_length) + kFewGranule - 1) / kFewGranule);
  }
  return f;
}

// CTAs that share `total` granules: every one of them gets at least one.
KIB_DEV int64_t few_ctas(int64_t total, int64_t grid) { return total < grid ? total : grid; }

template <int HD, int NT>
constexpr int few_partial_floats() { return 8 * NT * (HD + 2); }
template <int HD>
constexpr int few_ctas_per_sm() { return HD == 256 ? 1 : (HD == 128 ? 2 : 3); }
template <typename T, int HD, int NT>
constexpr size_t few_smem() {
  constexpr int planes = sizeof(T) == 4 ? 2 : 1;
  return static_cast<size_t>(8 * NT) * planes * (HD * 2 + 16) + static_cast<size_t>(kFewWarps) * 8 * NT * (HD + 4) * 4;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kFewWarps * 32, few_ctas_per_sm<HD>())
    kvq8_few_kernel(const __grid_constant__ Kvq8AttnParams p) {
  constexpr int RG = 8 * NT;                      // rows of a unit
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;      // half planes of q and p
  constexpr int QB = HD * 2 + 16;                 // bytes of a q row: conflict-free 16-byte reads
  constexpr int OF = HD + 4;                      // floats of an O row in shared memory
  constexpr int KL = HD / 64, VL = HD / 128 > 0 ? HD / 128 : 1;
  extern __shared__ __align__(16) uint8_t few_raw[];
  uint8_t* s_q = few_raw;                                           // [PL][RG][QB]
  float* s_o = reinterpret_cast<float*>(few_raw + PL * RG * QB);    // [warps][RG][OF]
  __shared__ int64_t s_cum[kFewMaxSeqs + 1];
  __shared__ int64_t s_warp[kFewWarps];
  __shared__ float s_qs[RG], s_m[kFewWarps][RG], s_l[kFewWarps][RG];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int S = p.b.sequences, kvh = p.c.kv_heads;

  // running granule totals of the sequences
  int64_t base = 0;
  for (int s0 = 0; s0 < S; s0 += kFewWarps * 32) {
    const int s = s0 + tid;
    int64_t v = 0;
    if (s < S) {
      const FewSeq f = few_seq<NT>(p, s);
      v = static_cast<int64_t>(f.granules) * f.groups * kvh;
    }
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int64_t before = base;
    for (int w = 0; w < kFewWarps; ++w) {
      if (w < warp) before += s_warp[w];
      base += s_warp[w];
    }
    if (s < S) s_cum[s] = before + inc - v;
    __syncthreads();
  }
  if (tid == 0) s_cum[S] = base;
  __syncthreads();
  const int64_t total = base;
  const int64_t ctas = few_ctas(total, gridDim.x);
  if (blockIdx.x >= ctas) return;
  int64_t at = total * blockIdx.x / ctas;
  const int64_t stop = total * (blockIdx.x + 1) / ctas;
  const int64_t first = at;
  int seq;
  {
    int lo = 0, hi = S;  // the last sequence that begins at or before `at`
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cum[mid] <= at) lo = mid;
      else hi = mid;
    }
    seq = lo;
  }

  while (at < stop) {
    while (s_cum[seq + 1] <= at) ++seq;
    const Kvq8Seq sq = kvq8_seq(p.b, seq);
    const FewSeq fs = few_seq<NT>(p, seq);
    const int64_t rel = at - s_cum[seq];
    const int unit = static_cast<int>(rel / fs.granules), gran0 = static_cast<int>(rel % fs.granules);
    const int head = unit % kvh, rg = unit / kvh;
    const int gran1 = static_cast<int>(min(static_cast<int64_t>(fs.granules), gran0 + (stop - at)));
    const int64_t begin = at;
    at += gran1 - gran0;
    const int64_t nrows = static_cast<int64_t>(sq.n) * p.group;
    const int row0 = rg * RG, live = static_cast<int>(min(static_cast<int64_t>(RG), nrows - row0));
    const int start = sq.length - sq.n;  // position of the first row
    const int span = max(0, min(sq.length, p.b.max_length));
    const int key0 = gran0 * kFewGranule;
    const int key1 = min(min(span, gran1 * kFewGranule), start + (row0 + live - 1) / p.group + 1);
    const int all_see = start + row0 / p.group + 1;  // keys below it are seen by every row

    // q rows to shared memory, as halves (fp32 rows scaled to about 2^13 by a power of two first)
    __syncthreads();
    for (int r = warp; r < RG; r += kFewWarps) {
      constexpr int V = HD / 32;
      float x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = 0.0f;
      if (r < live) {
        const int row = row0 + r;
        load_vec<T, V>(static_cast<const T*>(p.q) + static_cast<int64_t>(sq.first + row / p.group) * p.q_stride +
                           (static_cast<int64_t>(head) * p.group + row % p.group) * HD + lane * V,
                       x);
      }
      float back = 1.0f;
      if constexpr (PL == 2) {
        float big = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) big = fmaxf(big, fabsf(x[e]));
        big = warp_max(big);
        const int ex = static_cast<int>(__float_as_uint(big) >> 23);  // 255: not finite
        if (ex > 20 && ex < 255) {
          const int k = min(max(140 - ex, -100), 100);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
          back = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] *= up;
        }
      }
      alignas(16) __half hi[V], lo[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        hi[e] = __float2half_rn(x[e]);
        lo[e] = __float2half_rn(x[e] - __half2float(hi[e]));
      }
      uint8_t* dst = s_q + r * QB + lane * V * 2;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        *reinterpret_cast<__half2*>(dst + 2 * e) = __halves2half2(hi[e], hi[e + 1]);
        if constexpr (PL == 2) *reinterpret_cast<__half2*>(dst + RG * QB + 2 * e) = __halves2half2(lo[e], lo[e + 1]);
      }
      if (lane == 0) s_qs[r] = back * p.scale_log2;
    }
    __syncthreads();

    float o[HD / 16][NT][4];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.0f;
    float m[NT][2], l[NT][2], qs[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) m[j][e] = -INFINITY, l[j][e] = 0.0f, qs[j][e] = s_qs[8 * j + 2 * c + e];
    int vexp = 20;  // exponent field of the power of two that p is relative to

    uint4 kr[KL][2], vr[VL][4];
    float ks = 0.0f, vs = 0.0f, ks_n = 0.0f, vs_n = 0.0f;
    const int kstep = kFewWarps * 16;
    int key = key0 + warp * 16;
    auto page_at = [&](int k) { return k < key1 ? kvq8_page(p.c, p.b, seq, k >> p.c.page_shift) : -1; };
    auto tile = [&](const int8_t* codes, int page, int k) {
      return codes + page * p.c.page_stride + head * p.c.head_stride + (k & (p.c.page_tokens - 1)) * p.c.token_stride;
    };
    auto load_k = [&](int page, int k) {
      if (page < 0) return;
      const int8_t* t = tile(p.c.k, page, k) + 16 * c;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KL; ++i) kr[i][h] = ldg_stream(t + (g + 8 * h) * p.c.token_stride + 64 * i);
      const int64_t at_s = static_cast<int64_t>(page) * kvh + head;
      ks_n = __ldg(p.c.k_scale + at_s);
      vs_n = __ldg(p.c.v_scale + at_s);
    };
    int page = page_at(key), page_n = page_at(key + kstep);
    load_k(page, key);
    for (; key < key1; key += kstep) {
      const int page_nn = page_at(key + 2 * kstep);
      ks = ks_n, vs = vs_n;
      if (page >= 0) {
        const int8_t* t = tile(p.c.v, page, key);
        if constexpr (HD >= 128) {
#pragma unroll
          for (int i = 0; i < VL; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vr[i][e] = ldg_stream(t + (2 * c + (e & 1) + 8 * (e >> 1)) * p.c.token_stride + 128 * i + 16 * g);
        } else {
          // 64 dimensions: 8 bytes a lane and key
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(t + (2 * c + (e & 1) + 8 * (e >> 1)) * p.c.token_stride + 8 * g));
            vr[0][e].x = x.x, vr[0][e].y = x.y;
          }
        }
        float sc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const uint32_t w0[4] = {kr[i][0].x ^ 0x80808080u, kr[i][0].y ^ 0x80808080u, kr[i][0].z ^ 0x80808080u,
                                  kr[i][0].w ^ 0x80808080u};
          const uint32_t w1[4] = {kr[i][1].x ^ 0x80808080u, kr[i][1].y ^ 0x80808080u, kr[i][1].z ^ 0x80808080u,
                                  kr[i][1].w ^ 0x80808080u};
          uint4 qf[PL][NT][2];
#pragma unroll
          for (int pl = 0; pl < PL; ++pl)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint4* src = reinterpret_cast<const uint4*>(s_q + (pl * RG + 8 * j + g) * QB + 128 * i + 32 * c);
              qf[pl][j][0] = src[0];
              qf[pl][j][1] = src[1];
            }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t a0 = codes_to_half2(w0[u], 0x4140u), a2 = codes_to_half2(w0[u], 0x4342u);
            const uint32_t a1 = codes_to_half2(w1[u], 0x4140u), a3 = codes_to_half2(w1[u], 0x4342u);
#pragma unroll
            for (int pl = 0; pl < PL; ++pl)
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                const uint4 qv = qf[pl][j][u >> 1];
                mma_16816(sc[j], a0, a1, a2, a3, u & 1 ? qv.z : qv.x, u & 1 ? qv.w : qv.y);
              }
          }
        }
        load_k(page_n, key + kstep);

        // softmax over the tile's keys g and g + 8
        const bool edge = key + 16 > all_see || key + 16 > key1;
        const int ve = min(max(static_cast<int>(__float_as_uint(vs) >> 23), 20), 254);
        const float kmul = ks;
        float mn[NT][2];
        bool grow = ve > vexp;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mul = kmul * qs[j][e];
            float a = sc[j][e] * mul, b = sc[j][e + 2] * mul;
            if (edge) {
              const int r = 8 * j + 2 * c + e;
              const int end = r < live ? min(key1, start + (row0 + r) / p.group + 1) : 0;
              if (key + g >= end) a = -INFINITY;
              if (key + g + 8 >= end) b = -INFINITY;
            }
            sc[j][e] = a, sc[j][e + 2] = b;
            float t2 = fmaxf(a, b);
            t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, 4));
            t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, 8));
            t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, 16));
            mn[j][e] = fmaxf(m[j][e], t2);
            grow = grow || mn[j][e] > m[j][e];
          }
        if (__any_sync(0xffffffffu, grow)) {
          const int vn = max(ve, vexp);
          const float vf = __uint_as_float(static_cast<uint32_t>(max(127 + vexp - vn, 0)) << 23);
          vexp = vn;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = m[j][e] == -INFINITY ? 0.0f : ex2(m[j][e] - mn[j][e]);
              m[j][e] = mn[j][e];
              l[j][e] *= f;
              const float fo = f * vf;
#pragma unroll
              for (int i = 0; i < HD / 16; ++i) o[i][j][e] *= fo, o[i][j][e + 2] *= fo;
            }
        }
        // 2^14 * v_scale / 2^(vexp - 126)
        const float vmul = vs * __uint_as_float(static_cast<uint32_t>(min(127 + 140 - vexp, 254)) << 23);
        uint32_t pb[PL][NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mm = fmaxf(m[j][e], -1e30f);
            const float a = ex2(sc[j][e] - mm), b = ex2(sc[j][e + 2] - mm);
            l[j][e] += a + b;
            w[e] = a * vmul;
            w[e + 2] = b * vmul;
          }
          const uint32_t h0 = pack_half2(w[0], w[1]), h1 = pack_half2(w[2], w[3]);
          pb[0][j][0] = transpose_8x8(h0);
          pb[0][j][1] = transpose_8x8(h1);
          if constexpr (PL == 2) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
            pb[PL - 1][j][0] = transpose_8x8(pack_half2(w[0] - f0.x, w[1] - f0.y));
            pb[PL - 1][j][1] = transpose_8x8(pack_half2(w[2] - f1.x, w[3] - f1.y));
          }
        }
        // O^T += V^T P^T
        constexpr int WORDS = HD >= 128 ? 4 : 2;
#pragma unroll
        for (int i = 0; i < VL; ++i)
#pragma unroll
          for (int u = 0; u < WORDS; ++u) {
            const uint32_t x0 = u == 0 ? vr[i][0].x : u == 1 ? vr[i][0].y : u == 2 ? vr[i][0].z : vr[i][0].w;
            const uint32_t x1 = u == 0 ? vr[i][1].x : u == 1 ? vr[i][1].y : u == 2 ? vr[i][1].z : vr[i][1].w;
            const uint32_t x2 = u == 0 ? vr[i][2].x : u == 1 ? vr[i][2].y : u == 2 ? vr[i][2].z : vr[i][2].w;
            const uint32_t x3 = u == 0 ? vr[i][3].x : u == 1 ? vr[i][3].y : u == 2 ? vr[i][3].z : vr[i][3].w;
            const uint32_t lo01 = prmt(x0, x1, 0x5140u) ^ 0x80808080u, hi01 = prmt(x0, x1, 0x7362u) ^ 0x80808080u;
            const uint32_t lo23 = prmt(x2, x3, 0x5140u) ^ 0x80808080u, hi23 = prmt(x2, x3, 0x7362u) ^ 0x80808080u;
            const uint32_t a0 = codes_to_half2(lo01, 0x4140u), a1 = codes_to_half2(lo01, 0x4342u);
            const uint32_t a2 = codes_to_half2(lo23, 0x4140u), a3 = codes_to_half2(lo23, 0x4342u);
            const uint32_t c0 = codes_to_half2(hi01, 0x4140u), c1 = codes_to_half2(hi01, 0x4342u);
            const uint32_t c2 = codes_to_half2(hi23, 0x4140u), c3 = codes_to_half2(hi23, 0x4342u);
            const int mt = (i * WORDS + u) * 2;
#pragma unroll
            for (int pl = 0; pl < PL; ++pl)
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma_16816(o[mt][j], a0, a1, a2, a3, pb[pl][j][0], pb[pl][j][1]);
                mma_16816(o[mt + 1][j], c0, c1, c2, c3, pb[pl][j][0], pb[pl][j][1]);
              }
          }
      } else {
        load_k(page_n, key + kstep);
      }
      page = page_n;
      page_n = page_nn;
    }

    // join the warps: common maximum, then sums in warp order
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t2 = l[j][e];
        t2 += __shfl_xor_sync(0xffffffffu, t2, 4);
        t2 += __shfl_xor_sync(0xffffffffu, t2, 8);
        t2 += __shfl_xor_sync(0xffffffffu, t2, 16);
        if (g == 0) s_m[warp][8 * j + 2 * c + e] = m[j][e], s_l[warp][8 * j + 2 * c + e] = t2;
      }
    const float back = __uint_as_float(static_cast<uint32_t>(max(vexp - 13, 1)) << 23);  // 2^(vexp - 126 - 14)
    float* mine = s_o + warp * RG * OF;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(mine + (8 * j + 2 * c + e) * OF + (i * 8 + g) * 2) =
              make_float2(o[i][j][e] * back, o[i][j][e + 2] * back);
    __syncthreads();
    const bool whole = gran0 == 0 && gran1 == fs.granules;
    float* rec = nullptr;
    if (!whole) rec = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (begin == first ? 0 : 1)) * few_partial_floats<HD, NT>();
    for (int r = warp; r < live; r += kFewWarps) {
      float top = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kFewWarps; ++w) top = fmaxf(top, s_m[w][r]);
      float f[kFewWarps], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        f[w] = s_m[w][r] == -INFINITY ? 0.0f : ex2(s_m[w][r] - top);
        sum += f[w] * s_l[w][r];
      }
      const float inv = whole ? (sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum)) : 1.0f;
      const int row = row0 + r;
      constexpr int V = HD / 32;
      float x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int d = lane * V + e;
        // where dimension d lies: lane g and fragment i of the loads above
        constexpr int PER = HD >= 128 ? 16 : 8, SLAB = HD >= 128 ? 128 : 64;
        const int in = d % SLAB;
        const int idx = (((d / SLAB) * (PER / 2) + (in % PER) / 2) * 8 + in / PER) * 2 + (d & 1);
        float acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) acc += f[w] * s_o[(w * RG + r) * OF + idx];
        x[e] = acc * inv;
      }
      if (whole) {
        store_vec<T, V>(static_cast<T*>(p.out) + static_cast<int64_t>(sq.first + row / p.group) * p.out_stride +
                            (static_cast<int64_t>(head) * p.group + row % p.group) * HD + lane * V,
                        x);
      } else {
        store_vec<float, V>(rec + r * HD + lane * V, x);
        if (lane == 0) rec[RG * HD + 2 * r] = top, rec[RG * HD + 2 * r + 1] = sum;
      }
    }
  }
}

// Joins the records of the units that cross CTAs, in CTA order.  One CTA per
// (row of a unit, unit); most find a whole unit and leave.
constexpr int kMergeMaxCtas = 1024;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(HD) kvq8_merge_kernel(const __grid_constant__ Kvq8AttnParams p, int grid_ctas, int max_groups) {
  constexpr int RG = 8 * NT, W = HD / 32;
  __shared__ int64_t s_sum[2][W];
  __shared__ float s_f[kMergeMaxCtas], s_red[2][W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.y, kvh = p.c.kv_heads;
  const int head = blockIdx.x % kvh, rg = blockIdx.x / kvh % max_groups, seq = blockIdx.x / kvh / max_groups;
  // the batch's description is not this launch's predecessor's work: read it before the wait
  const FewSeq fs = few_seq<NT>(p, seq);
  const Kvq8Seq sq = kvq8_seq(p.b, seq);
  const int64_t row = static_cast<int64_t>(rg) * RG + r;
  // every CTA waits before it leaves: a grid that ends early would let the
  // stream's next kernel run beside the one before this
  if (rg >= fs.groups || row >= static_cast<int64_t>(sq.n) * p.group) {
    pdl_wait();
    return;
  }
  int64_t before = 0, total = 0;
  for (int s = tid; s < p.b.sequences; s += HD) {
    const FewSeq f = few_seq<NT>(p, s);
    const int64_t v = static_cast<int64_t>(f.granules) * f.groups * kvh;
    total += v;
    if (s < seq) before += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) s_sum[0][warp] = before, s_sum[1][warp] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) before += s_sum[0][w], total += s_sum[1][w];
  const int64_t lo = before + static_cast<int64_t>(rg * kvh + head) * fs.granules, hi = lo + fs.granules;
  const int64_t ctas = few_ctas(total, grid_ctas);
  // CTA i holds [total * i / ctas, total * (i + 1) / ctas): the one of granule x
  auto owner = [&](int64_t x) {
    int64_t i = x * ctas / total;
    while (total * (i + 1) / ctas <= x) ++i;
    while (total * i / ctas > x) --i;
    return static_cast<int>(i);
  };
  const int c0 = owner(lo), n = owner(hi - 1) - c0 + 1;
  pdl_wait();
  if (n == 1) return;
  // a CTA's first run is its record 0: the unit's, but where the unit begins inside the CTA
  constexpr int64_t REC = few_partial_floats<HD, NT>();
  const float* rec0 = p.partial + static_cast<int64_t>(c0) * 2 * REC;
  const float* rec_first = rec0 + (total * c0 / ctas < lo ? REC : 0);
  float top = -INFINITY;
  for (int i = tid; i < n; i += HD) {
    const float m = (i ? rec0 + 2 * REC * i : rec_first)[RG * HD + 2 * r];
    s_f[i] = m;
    top = fmaxf(top, m);
  }
  top = warp_max(top);
  if (lane == 0) s_red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, s_red[0][w]);
  float sum = 0.0f;
  for (int i = tid; i < n; i += HD) {
    const float f = s_f[i] == -INFINITY ? 0.0f : ex2(s_f[i] - top);
    s_f[i] = f;
    sum += f * (i ? rec0 + 2 * REC * i : rec_first)[RG * HD + 2 * r + 1];
  }
  sum = warp_sum(sum);
  if (lane == 0) s_red[1][warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) sum += s_red[1][w];
  float acc = s_f[0] * rec_first[r * HD + tid];
#pragma unroll 8
  for (int i = 1; i < n; ++i) acc += s_f[i] * rec0[2 * REC * i + r * HD + tid];
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  T* out = static_cast<T*>(p.out) + static_cast<int64_t>(sq.first + row / p.group) * p.out_stride +
           (static_cast<int64_t>(head) * p.group + row % p.group) * HD;
  out[tid] = from_f32<T>(acc * inv);
}

}  // namespace kib
