// kvq8_few.cuh -- attention of few rows per sequence (single decoded tokens,
// speculative verify) over the paged 8-bit cache.
//
// For a unit (sequence, KV head, group of up to 8 NT query rows) the cache's
// codes pass once through registers:
//   S^T = K Q^T, s = S * k_scale * scale, reference m, p = 2^(s - m),
//   O^T += V^T (p * v_scale)^T, l += p;   out = O / l.
// m is a score of the row that no later one exceeds by more than 2^8: only
// when one does (a vote, no reduction) is the true maximum taken and O
// rescaled.  Codes are integers below 128 in magnitude, exact in half, so only
// q and p are rounded: half rows use q as given and p as one half; fp32 rows
// use both as high + low halves (22 bits).  v_scale goes into p, relative to
// the largest power of two met so far (exact to move) and 2^7 above it: p
// stays below 2^15 and keeps its accuracy in half down to 2^-21 of a weight
// of one (with the low half to 2^-31).
//
// Work is cut into granules of 128 keys, laid end to end over all units; each
// of the grid's CTAs takes an equal run of them, whatever the lengths are, so
// the kernel needs no host knowledge of the lengths.  A unit that crosses
// CTAs leaves partial (m, l, O) records, which kvq8_merge_kernel joins in
// order: the result depends on no timing.  Within a CTA, the warps take
// tiles of 16 to 64 keys in turn, each with its own m, l and O, and join in shared
// memory at the end of the unit's run.
//
// Bound by HBM: 2 bytes per key, head and dimension, and next by the
// instructions that unpack them.  Every warp has a ring of tiles of its own in
// shared memory that one of its lanes refills by tensor-map TMA over the
// cache's own layout (any strides): a K or V piece is asked for as soon as its
// predecessor has been read, so no register and no other warp waits for a
// load; the pages and scales of the warp's next 32 tiles sit in its lanes.
// (One producer warp serving all others, a lane each, kept up with 4.4 TB/s
// only: its TMA instructions issue one lane after another.)  The 128-byte
// swizzle keeps both fragment reads free of bank conflicts: a lane's 16 bytes
// of a K row are the A fragments of four mma k-steps (the dimensions of a dot
// product may be taken in any order, and q is laid out the same way); of V,
// two byte permutes transpose 4 keys x 2 dimensions into a fragment.
// Measured, 2 KV heads of 256 with 4 query heads each: 64 sequences of up to
// 32768, half rows: 209-217 us, 6.2 to 6.5 TB/s; 32 of about 2048, fp32: 26.5 us;
// one of 4096: 13 us.  17 sequences of up to 8190 with up to 5 fp32 rows each
// of 16 heads of 128: 54.5 us, 1.5 TB/s, where three groups of rows with two
// halves of q and of p leave more instructions a key than bytes.
#pragma once

#include "gemm_tc.cuh"
#include "kvq8.cuh"

namespace kib {

constexpr int kFewGranule = 128;
// A run takes about 4.5 us besides its granules (pages looked up, q in, the
// first tiles awaited, the warps joined), what an SM's share of the memory's
// rate moves in three granules of 256 dimensions: runs are cut by granules
// plus this, so that few CTAs get two.  (32 slots of about 2048: 24.8 us
// without it, 27.9 with 8; verify of 17 sequences at 128 dimensions: 58.6 us
// without it, 51.5 with 8.)
__host__ __device__ constexpr int few_unit_cost(int hd) { return 768 / hd; }
constexpr int kFewMaxSeqs = 4096;

// Warps of a CTA (one CTA per SM), by what the accumulators (head_dim / 16 x
// NT x 4 registers a lane) leave.
__host__ __device__ constexpr int few_warps_of(int hd, int nt) { return hd / 16 * nt * 4 >= 96 ? 8 : 12; }
template <int HD, int NT>
constexpr int few_warps() { return few_warps_of(HD, NT); }
// A warp's tile: this many blocks of 16 keys, 2 or 4 KB of K and as much of V.
__host__ __device__ constexpr int few_blocks(int hd) { return hd == 256 ? 1 : 2; }
// Tiles in a warp's ring, within 192 KB for all warps.
template <int HD, int NT>
constexpr int few_ring() {
  constexpr int n = 196608 / (few_warps<HD, NT>() * 32 * HD * few_blocks(HD));
  return n < 4 ? n : 4;
}
// The MMA's fp32 sums are cut toward zero, up to an ulp at every step: a chain
// of them over 32768 keys would be off by 3.9e-6 of a random result, by 33e-6 where
// one key holds the weight and all V are alike.  So a tile of fp32 rows is
// summed from zero, low halves first, and added to O with rounding; l takes
// along what its additions round off (after one key of weight 1, the rest may
// be smaller than l's last bit); and where a tile is 16 keys only, O moves into
// sums in memory every kFewBank tiles, so that a long tail of small tiles is
// not rounded off either.  Error then: 0.1e-6 to 0.6e-6 of the result.  Cost:
// 32 slots of about 2048 24.5 -> 26.7 us, verify 49.4 -> 54.5 us, 64 sequences
// to 32768 with fp32 rows 229 -> 266 us (without the moves 258).
constexpr int kFewBank = 64;  // tiles
template <typename T>
__host__ __device__ constexpr bool few_banks(int hd) { return sizeof(T) == 4 && few_blocks(hd) == 1; }
// Groups of 8 rows a unit may have.
__host__ __device__ constexpr int few_max_nt(int hd) { return hd == 256 ? 2 : 3; }

struct Kvq8AttnParams {
  Kvq8Cache c;
  Kvq8Batch b;
  const void* q;
  void* out;
  int heads, group;  // group = heads / kv_heads
  int64_t q_stride, out_stride;
  float scale_log2;  // softmax scale times log2(e)
  float* partial;    // [ctas][2][rows of a unit][head_dim + 2]
  float4* bank;      // fp32 rows: [ctas][warps][head_dim / 16][groups of 8 rows][32 lanes] sums that O moves into
  int few_limit;     // sequences of at most this many rows * group are this kernel's
  int* err;
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
// The same onto zeros.
KIB_DEV void mma_16816_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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

KIB_DEV void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// store_vec where a lane may hold a single value.
template <typename T, int V>
KIB_DEV void store_any(T* p, const float (&x)[V]) {
  if constexpr (V * sizeof(T) >= 4) store_vec<T, V>(p, x);
  else p[0] = from_f32<T>(x[0]);
}

// Granules of one unit of a sequence, and its units per KV head.
struct FewSeq {
  int granules, groups, unit;
  KIB_DEV int64_t cost() const { return granules + unit; }
};
template <int HD, int NT>
KIB_DEV FewSeq few_seq(const Kvq8AttnParams& p, int s) {
  const Kvq8Seq q = kvq8_seq(p.b, s);
  const int64_t rows = static_cast<int64_t>(q.n) * p.group;
  FewSeq f{0, 0, few_unit_cost(HD)};
  if (q.n > 0 && rows <= p.few_limit) {
    f.groups = static_cast<int>((rows + 8 * NT - 1) / (8 * NT));
    f.granules = max(1, (min(q.length, p.b.max_length) + kFewGranule - 1) / kFewGranule);
  }
  return f;
}

// CTAs that share a cost of `total`: every one of them gets at least one.
KIB_DEV int64_t few_ctas(int64_t total, int64_t grid) { return total < grid ? total : grid; }

template <int HD, int NT>
constexpr int few_partial_floats() { return 8 * NT * (HD + 2); }
template <typename T, int HD, int NT>
constexpr size_t few_smem() {
  constexpr int planes = sizeof(T) == 4 ? 2 : 1, warps = few_warps<HD, NT>();
  constexpr size_t ring = static_cast<size_t>(warps) * few_ring<HD, NT>() * 32 * HD * few_blocks(HD);
  constexpr size_t join = static_cast<size_t>(warps) * 8 * NT * (HD + 4) * 4;
  return (ring > join ? ring : join) + static_cast<size_t>(8 * NT) * planes * (HD * 2 + 16);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(few_warps<HD, NT>() * 32, 1)
    kvq8_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ Kvq8AttnParams p) {
  constexpr int RG = 8 * NT;                      // rows of a unit
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;      // half planes of q and p
  constexpr int QB = HD * 2 + 16;                 // bytes of a q row: conflict-free 16-byte reads
  constexpr int OF = HD + 4;                      // floats of an O row in shared memory
  constexpr bool BANK = few_banks<T>(HD);         // O moves into sums in memory now and then
  constexpr int W = few_warps<HD, NT>(), D = few_ring<HD, NT>(), MK = few_blocks(HD), BLOCK = 16 * HD, PIECE = MK * BLOCK;
  constexpr size_t RING = static_cast<size_t>(W) * D * 2 * PIECE, JOIN = static_cast<size_t>(W) * RG * OF * 4;
  extern __shared__ __align__(1024) uint8_t few_raw[];
  float* s_o = reinterpret_cast<float*>(few_raw);                   // [W][RG][OF], in the ring's place once it is empty
  uint8_t* s_q = few_raw + (RING > JOIN ? RING : JOIN);             // [PL][RG][QB]
  __shared__ uint64_t s_bar[W][D][2];                               // K and V of a ring slot have arrived
  __shared__ int64_t s_warp[W], s_at;
  __shared__ int s_seq;
  __shared__ float s_qs[RG], s_m[W][RG], s_l[W][RG];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int S = p.b.sequences, kvh = p.c.kv_heads;
  if (lane < 2 * D) mbar_init(&s_bar[warp][lane >> 1][lane & 1], 1);
  fence_mbar_init();
  if (tid == 0) tma_prefetch_desc(&kmap), tma_prefetch_desc(&vmap);

  pdl_launch_dependents();  // the merge's CTAs may take the SMs that are left and wait there

  // the cost of all sequences; then the sequence in which this CTA's run begins
  constexpr int TH = W * 32;
  auto seq_cost = [&](int s) -> int64_t {
    if (s >= S) return 0;
    const FewSeq f = few_seq<HD, NT>(p, s);
    return f.cost() * f.groups * kvh;
  };
  auto scan = [&](int64_t v, int64_t* all) {
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += s_warp[w];
      sum += s_warp[w];
    }
    *all = sum;
    return before + inc - v;
  };
  const int64_t cost0 = seq_cost(tid);
  int64_t all0;
  const int64_t x0 = scan(cost0, &all0);
  int64_t total = all0;
  for (int s0 = TH; s0 < S; s0 += TH) {
    int64_t all;
    scan(seq_cost(s0 + tid), &all);
    total += all;
  }
  const int64_t ctas = few_ctas(total, gridDim.x);
  if (blockIdx.x >= ctas) return;
  int64_t at = total * blockIdx.x / ctas;
  const int64_t stop = total * (blockIdx.x + 1) / ctas, first = at;
  if (x0 <= at && at < x0 + cost0) s_seq = tid, s_at = x0;
  int64_t base = all0;
  for (int s0 = TH; s0 < S && base <= at; s0 += TH) {
    int64_t all;
    const int64_t v = seq_cost(s0 + tid), x = base + scan(v, &all);
    if (x <= at && at < x + v) s_seq = s0 + tid, s_at = x;
    base += all;
  }
  __syncthreads();
  int seq = s_seq;
  int64_t seq_at = s_at;  // cost before the sequence

  // the run of granules [gran0, gran1) of a unit that begins at `at`
  struct Run {
    Kvq8Seq sq;
    int head, row0, live, key0, key1;
    bool whole, empty;
  };
  auto next_run = [&]() {
    Run r;
    r.sq = kvq8_seq(p.b, seq);
    FewSeq fs = few_seq<HD, NT>(p, seq);
    while (at >= seq_at + fs.cost() * fs.groups * kvh) {
      seq_at += fs.cost() * fs.groups * kvh;
      ++seq;
      r.sq = kvq8_seq(p.b, seq);
      fs = few_seq<HD, NT>(p, seq);
    }
    const int64_t rel = at - seq_at;
    const int unit = static_cast<int>(rel / fs.cost());
    const int64_t g0 = rel - unit * fs.cost() - few_unit_cost(HD), g1 = min(static_cast<int64_t>(fs.granules), g0 + (stop - at));
    const int gran0 = static_cast<int>(max(g0, static_cast<int64_t>(0))), gran1 = static_cast<int>(max(g1, static_cast<int64_t>(0)));
    r.head = unit % kvh;
    r.row0 = unit / kvh * RG;
    r.live = min(RG, r.sq.n * p.group - r.row0);
    r.key0 = gran0 * kFewGranule;
    const int span = max(0, min(r.sq.length, p.b.max_length));
    r.key1 = min(min(span, gran1 * kFewGranule), r.sq.length - r.sq.n + (r.row0 + r.live - 1) / p.group + 1);
    r.whole = gran0 == 0 && gran1 == fs.granules;
    r.empty = gran0 == gran1;
    at += g1 - g0;
    return r;
  };

  uint32_t slot_i = 0, slot = 0, phase = 0;  // ring slots: of the next tile to ask for, and to work on
  bool ok = true;
  uint8_t* ring = few_raw + static_cast<size_t>(warp) * D * 2 * PIECE;
  while (at < stop) {
    const int64_t begin = at;
    const Run r = next_run();
    if (r.empty) continue;
    const Kvq8Seq sq = r.sq;
    const int head = r.head, row0 = r.row0, live = r.live, key1 = r.key1, start = sq.length - sq.n;
    const int all_see = start + row0 / p.group + 1;  // keys below it are seen by every row

    // this warp's tiles: keys from key0 + 16 MK (warp + W t) on; lane b % 32 holds the page and scales of block b
    const int first_key = r.key0 + 16 * MK * warp;
    const int tiles = key1 > first_key ? (key1 - first_key - 1) / (16 * MK * W) + 1 : 0;
    auto block_key = [&](int b) { return first_key + 16 * MK * W * (b / MK) + 16 * (b % MK); };
    auto lane_page = [&](int b0) {
      const int key = block_key(b0 + lane);
      return key < key1 ? kvq8_page(p.c, p.b, seq, key >> p.c.page_shift) : -1;
    };
    auto lane_scale = [&](const float* s, int page) { return page >= 0 ? __ldg(s + static_cast<int64_t>(page) * kvh + head) : 0.0f; };
    int page_l = lane_page(0), page_n = lane_page(32), page_nn = -1;  // of this batch of 32 blocks, the next and its next
    int batch = 0;                // the first block of the batch in the lanes
    int ti = 0, page_i[MK] = {};  // the next tile to ask for; the pages of the one whose K was asked for last
    // what is absent or past the run is neither copied nor looked at (its weights are 0, and codes are numbers)
    auto piece = [&](const CUtensorMap* map, int half, int tile) {
      if (lane == 0) {
        uint64_t* bar = &s_bar[warp][slot_i][half];
        uint8_t* dst = ring + (slot_i * 2 + half) * PIECE;
        int bytes = 0;
#pragma unroll
        for (int b = 0; b < MK; ++b) bytes += page_i[b] >= 0 ? BLOCK : 0;
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int b = 0; b < MK; ++b) {
          if (page_i[b] < 0) continue;
          const int row = block_key(tile * MK + b) & (p.c.page_tokens - 1);
#pragma unroll
          for (int i = 0; i < (HD + 127) / 128; ++i)
            tma_load_4d(dst + b * BLOCK + 2048 * i, map, 128 * i, row, head, page_i[b], bar);
        }
      }
    };
    auto ask_k = [&]() {
      if (ti >= tiles) return;
#pragma unroll
      for (int b = 0; b < MK; ++b)
        page_i[b] = __shfl_sync(0xffffffffu, ti * MK < batch + 32 ? page_l : page_n, (ti * MK + b) & 31);
      piece(&kmap, 0, ti);
    };
    auto ask_v = [&]() {
      if (ti >= tiles) return;
      piece(&vmap, 1, ti);
      ++ti;
      slot_i = slot_i + 1 == D ? 0 : slot_i + 1;
    };
#pragma unroll 1
    for (int i = 0; i < D; ++i) ask_k(), ask_v();
    float ks_l = lane_scale(p.c.k_scale, page_l), vs_l = lane_scale(p.c.v_scale, page_l), ks_n = 0.0f, vs_n = 0.0f;

    // q rows to shared memory, as halves (fp32 rows scaled to about 2^13 by a power of two first)
    for (int rr = warp; rr < RG; rr += W) {
      constexpr int V = HD / 32;
      float x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = 0.0f;
      if (rr < live) {
        const int row = row0 + rr;
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
      // 16 dimensions of chunk 2 c + i of a 128-dimension slab go to place 4 i + c: lane c's k-steps
      const int d = lane * V, ch = d % 128 / 16;
      const int place = HD >= 128 ? d / 128 * 128 + ((ch & 1) * 4 + (ch >> 1)) * 16 + d % 16 : d;
      uint8_t* dst = s_q + rr * QB + place * 2;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        *reinterpret_cast<__half2*>(dst + 2 * e) = __halves2half2(hi[e], hi[e + 1]);
        if constexpr (PL == 2) *reinterpret_cast<__half2*>(dst + RG * QB + 2 * e) = __halves2half2(lo[e], lo[e + 1]);
      }
      if (lane == 0) s_qs[rr] = back * p.scale_log2;
    }
    __syncthreads();

    float o[HD / 16][NT][4];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.0f;
    float m[NT][2], l[NT][2], lc[NT][2], qs[NT][2];  // lc: what the last addition to l rounded off (fp32 rows)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) m[j][e] = -INFINITY, l[j][e] = lc[j][e] = 0.0f, qs[j][e] = s_qs[8 * j + 2 * c + e];
    int vexp = 20;  // exponent field of the power of two that p is relative to

    // O's sums of long runs: bank = bank * 2^(what m and vexp grew by) + O (`into`), or O += that
    float m_bank[BANK ? NT : 1][2];  // m and vexp at the last move
    int vexp_bank = 0;               // 0: none yet
    auto bank = [&](bool into) {
      if constexpr (BANK) {
        float4* at_bank = p.bank + (static_cast<int64_t>(blockIdx.x) * W + warp) * (HD / 16 * NT * 32) + lane;
        float f[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float vf = __uint_as_float(static_cast<uint32_t>(max(127 + vexp_bank - vexp, 0)) << 23);
            f[j][e] = vexp_bank && m_bank[j][e] != -INFINITY ? ex2(m_bank[j][e] - m[j][e]) * vf : 0.0f;
            m_bank[j][e] = m[j][e];
          }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float (&x)[4] = o[i][j];
            if (vexp_bank) {
              const float4 s = at_bank[(i * NT + j) * 32];
              x[0] = fmaf(s.x, f[j][0], x[0]), x[1] = fmaf(s.y, f[j][1], x[1]);
              x[2] = fmaf(s.z, f[j][0], x[2]), x[3] = fmaf(s.w, f[j][1], x[3]);
            }
            if (into) {
              at_bank[(i * NT + j) * 32] = make_float4(x[0], x[1], x[2], x[3]);
              x[0] = x[1] = x[2] = x[3] = 0.0f;
            }
          }
        vexp_bank = vexp;
      }
    };

    auto wait_piece = [&](int half) { ok = ok && mbar_wait_bounded(&s_bar[warp][slot][half], phase, p.err); };
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      const int blk = t * MK;
      if (BANK && t % kFewBank == 0 && t) bank(true);
      if (blk == batch + 32) {
        batch = blk;
        page_l = page_n, page_n = page_nn;
        ks_l = ks_n, vs_l = vs_n;
      }
      // the batch after the next: its pages early in this one, the next one's scales later
      if (blk == batch + 4) page_nn = lane_page(batch + 64);
      if (blk == batch + 8) ks_n = lane_scale(p.c.k_scale, page_n), vs_n = lane_scale(p.c.v_scale, page_n);
      const int key = block_key(blk);
      float ks[MK], vs[MK];
      bool edge = key + 16 * MK > all_see || key + 16 * MK > key1;
      uint32_t gone = 0;  // blocks without a page
#pragma unroll
      for (int b = 0; b < MK; ++b) {
        ks[b] = __shfl_sync(0xffffffffu, ks_l, (blk + b) & 31), vs[b] = __shfl_sync(0xffffffffu, vs_l, (blk + b) & 31);
        if (__shfl_sync(0xffffffffu, page_l, (blk + b) & 31) < 0) gone |= 1u << b;
      }
      edge = edge || gone;
      wait_piece(0);

      // S^T = K Q^T; where one block has few accumulators, more of them keep the chains of dependent products short
      float sc[MK][NT][4];
      constexpr int SPLIT = MK * NT == 1 ? 2 * PL : (MK * NT == 2 ? PL : 1);
      {
        float sp[SPLIT][MK][NT][4];
#pragma unroll
        for (int a = 0; a < SPLIT; ++a)
#pragma unroll
          for (int b = 0; b < MK; ++b)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) sp[a][b][j][e] = 0.0f;
        const uint8_t* kt = ring + slot * 2 * PIECE;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
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
          for (int b = 0; b < MK; ++b) {
            // rows g and g + 8 share their swizzle
            const uint8_t* at_k = kt + b * BLOCK + (HD >= 128 ? 2048 * (i >> 1) + 128 * g + (((2 * c + (i & 1)) ^ g) << 4)
                                                              : 64 * g + ((c ^ (g >> 1)) << 4));
            const uint4 k0 = *reinterpret_cast<const uint4*>(at_k);
            const uint4 k1 = *reinterpret_cast<const uint4*>(at_k + (HD >= 128 ? 1024 : 512));
            const uint32_t w0[4] = {k0.x ^ 0x80808080u, k0.y ^ 0x80808080u, k0.z ^ 0x80808080u, k0.w ^ 0x80808080u};
            const uint32_t w1[4] = {k1.x ^ 0x80808080u, k1.y ^ 0x80808080u, k1.z ^ 0x80808080u, k1.w ^ 0x80808080u};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint32_t a0 = codes_to_half2(w0[u], 0x4140u), a2 = codes_to_half2(w0[u], 0x4342u);
              const uint32_t a1 = codes_to_half2(w1[u], 0x4140u), a3 = codes_to_half2(w1[u], 0x4342u);
#pragma unroll
              for (int pl = 0; pl < PL; ++pl)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                  const uint4 qv = qf[pl][j][u >> 1];
                  constexpr int A = SPLIT;
                  const int a = A == 1 ? 0 : (A == PL ? pl : 2 * pl + (u & 1));
                  mma_16816(sp[a][b][j], a0, a1, a2, a3, u & 1 ? qv.z : qv.x, u & 1 ? qv.w : qv.y);
                }
            }
          }
        }
#pragma unroll
        for (int b = 0; b < MK; ++b)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = sp[0][b][j][e];
#pragma unroll
              for (int a = 1; a < SPLIT; ++a) x += sp[a][b][j][e];
              sc[b][j][e] = x * (ks[b] * qs[j][e & 1]);
            }
      }
      __syncwarp();
      ask_k();

      // keys g and g + 8 of each block against the row's reference
      if (edge) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int rr = 8 * j + 2 * c + e;
            const int end = rr < live ? min(key1, start + (row0 + rr) / p.group + 1) : 0;
#pragma unroll
            for (int b = 0; b < MK; ++b) {
              const bool no = gone >> b & 1;
              if (no || key + 16 * b + g >= end) sc[b][j][e] = -INFINITY;
              if (no || key + 16 * b + g + 8 >= end) sc[b][j][e + 2] = -INFINITY;
            }
          }
      }
      int ve = 20;
#pragma unroll
      for (int b = 0; b < MK; ++b) ve = max(ve, min(static_cast<int>(__float_as_uint(vs[b]) >> 23), 254));
      bool grow = ve > vexp;
      float top[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[0][j][e], sc[0][j][e + 2]);
#pragma unroll
          for (int b = 1; b < MK; ++b) x = fmaxf(x, fmaxf(sc[b][j][e], sc[b][j][e + 2]));
          top[j][e] = x;
          grow = grow || x > m[j][e] + 8.0f;
        }
      if (__any_sync(0xffffffffu, grow)) {
        const int vn = max(ve, vexp);
        const float vf = __uint_as_float(static_cast<uint32_t>(max(127 + vexp - vn, 0)) << 23);
        vexp = vn;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[j][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float mn = fmaxf(m[j][e], x);
            const float f = m[j][e] == -INFINITY ? 0.0f : ex2(m[j][e] - mn);
            m[j][e] = mn;
            l[j][e] *= f, lc[j][e] *= f;
            const float fo = f * vf;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) o[i][j][e] *= fo, o[i][j][e + 2] *= fo;
          }
      }
      // 2^7 / 2^(vexp - 126)
      const float vup = __uint_as_float(static_cast<uint32_t>(min(260 - vexp, 254)) << 23);
      uint32_t pb[PL][MK][NT][2];
      float lt[NT][2] = {};
#pragma unroll
      for (int b = 0; b < MK; ++b) {
        const float vmul = vs[b] * vup;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mm = m[j][e] == -INFINITY ? 0.0f : m[j][e];
            const float x = ex2(sc[b][j][e] - mm), y = ex2(sc[b][j][e + 2] - mm);
            lt[j][e] += x + y;
            w[e] = x * vmul;
            w[e + 2] = y * vmul;
          }
          const uint32_t h0 = pack_half2(w[0], w[1]), h1 = pack_half2(w[2], w[3]);
          pb[0][b][j][0] = transpose_8x8(h0);
          pb[0][b][j][1] = transpose_8x8(h1);
          if constexpr (PL == 2) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
            pb[PL - 1][b][j][0] = transpose_8x8(pack_half2(w[0] - f0.x, w[1] - f0.y));
            pb[PL - 1][b][j][1] = transpose_8x8(pack_half2(w[2] - f1.x, w[3] - f1.y));
          }
        }
      }

#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (PL == 2) {
            const float y = __fsub_rn(lt[j][e], lc[j][e]), t2 = __fadd_rn(l[j][e], y);
            lc[j][e] = __fsub_rn(__fsub_rn(t2, l[j][e]), y);
            l[j][e] = t2;
          } else {
            l[j][e] += lt[j][e];
          }
        }

      // O^T += V^T P^T
      wait_piece(1);
      constexpr int WORDS = HD >= 128 ? 4 : 2, VL = HD >= 128 ? HD / 128 : 1;
      // half rows: block by block; fp32 rows: all blocks of the tile, low halves first, onto zeros, and these sums onto O
      constexpr int BB = PL == 2 ? MK : 1;
#pragma unroll
      for (int b0 = 0; b0 < MK; b0 += BB) {
#pragma unroll
        for (int i = 0; i < VL; ++i) {
          uint32_t x[BB][4][4];
#pragma unroll
          for (int b = 0; b < BB; ++b) {
            const uint8_t* vt = ring + (slot * 2 + 1) * PIECE + (b0 + b) * BLOCK;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = 2 * c + (e & 1) + 8 * (e >> 1);
              if constexpr (WORDS == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(vt + 2048 * i + 128 * row + ((g ^ (row & 7)) << 4));
                x[b][e][0] = v.x, x[b][e][1] = v.y, x[b][e][2] = v.z, x[b][e][3] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2*>(vt + 64 * row + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
                x[b][e][0] = v.x, x[b][e][1] = v.y;
              }
            }
          }
#pragma unroll
          for (int u = 0; u < WORDS; ++u) {
            uint32_t a[BB][2][4];  // fragments of 16 dimensions each
#pragma unroll
            for (int b = 0; b < BB; ++b) {
              const uint32_t lo01 = prmt(x[b][0][u], x[b][1][u], 0x5140u) ^ 0x80808080u, hi01 = prmt(x[b][0][u], x[b][1][u], 0x7362u) ^ 0x80808080u;
              const uint32_t lo23 = prmt(x[b][2][u], x[b][3][u], 0x5140u) ^ 0x80808080u, hi23 = prmt(x[b][2][u], x[b][3][u], 0x7362u) ^ 0x80808080u;
              a[b][0][0] = codes_to_half2(lo01, 0x4140u), a[b][0][1] = codes_to_half2(lo01, 0x4342u);
              a[b][0][2] = codes_to_half2(lo23, 0x4140u), a[b][0][3] = codes_to_half2(lo23, 0x4342u);
              a[b][1][0] = codes_to_half2(hi01, 0x4140u), a[b][1][1] = codes_to_half2(hi01, 0x4342u);
              a[b][1][2] = codes_to_half2(hi23, 0x4140u), a[b][1][3] = codes_to_half2(hi23, 0x4342u);
            }
            const int mt = (i * WORDS + u) * 2;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float (&d)[4] = o[mt + h][j];
                if constexpr (PL == 2) {
                  float t[4];
#pragma unroll
                  for (int b = 0; b < BB; ++b) {
                    if (b == 0) mma_16816_new(t, a[b][h][0], a[b][h][1], a[b][h][2], a[b][h][3], pb[1][b][j][0], pb[1][b][j][1]);
                    else mma_16816(t, a[b][h][0], a[b][h][1], a[b][h][2], a[b][h][3], pb[1][b][j][0], pb[1][b][j][1]);
                  }
#pragma unroll
                  for (int b = 0; b < BB; ++b) mma_16816(t, a[b][h][0], a[b][h][1], a[b][h][2], a[b][h][3], pb[0][b][j][0], pb[0][b][j][1]);
#pragma unroll
                  for (int e = 0; e < 4; ++e) d[e] += t[e];
                } else {
                  mma_16816(d, a[0][h][0], a[0][h][1], a[0][h][2], a[0][h][3], pb[0][b0][j][0], pb[0][b0][j][1]);
                }
              }
          }
        }
      }
      __syncwarp();
      ask_v();
      if (++slot == D) slot = 0, phase ^= 1;
    }

    if (BANK && vexp_bank) bank(false);

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
    const float back = __uint_as_float(static_cast<uint32_t>(max(vexp - 6, 1)) << 23);  // 2^(vexp - 126 - 7)
    __syncthreads();  // every ring is empty
    float* mine = s_o + warp * RG * OF;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (8 * j + 2 * c + e >= live || m[j][e] == -INFINITY) continue;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
          *reinterpret_cast<float2*>(mine + (8 * j + 2 * c + e) * OF + (i * 8 + g) * 2) =
              make_float2(o[i][j][e] * back, o[i][j][e + 2] * back);
      }
    __syncthreads();
    const bool whole = r.whole;
    float* rec = nullptr;
    if (!whole) rec = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (begin == first ? 0 : 1)) * few_partial_floats<HD, NT>();
    // a warp per row and part of the head, so that more warps work on few rows
    constexpr int PARTS = NT == 1 ? 2 : 1, V = HD / 32 / PARTS;
    for (int rp = warp; rp < live * PARTS; rp += W) {
      const int rr = rp / PARTS, d0 = (rp % PARTS) * (HD / PARTS) + lane * V;
      float top = s_m[0][rr];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, s_m[w][rr]);
      float sum = 0.0f, x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (s_m[w][rr] == -INFINITY) {
          sum += s_l[w][rr];  // 0: no key for this warp; NaN: scores that are no numbers, as the result then is
          continue;
        }
        const float f = ex2(s_m[w][rr] - top);
        sum += f * s_l[w][rr];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int d = d0 + e;
          // where dimension d lies: lane g and fragment i of the reads above
          constexpr int PER = HD >= 128 ? 16 : 8, SLAB = HD >= 128 ? 128 : 64;
          const int in = d % SLAB;
          const int idx = (((d / SLAB) * (PER / 2) + (in % PER) / 2) * 8 + in / PER) * 2 + (d & 1);
          x[e] += f * s_o[(w * RG + rr) * OF + idx];
        }
      }
      const int row = row0 + rr;
      if (whole) {
        const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= inv;
        store_any<T, V>(static_cast<T*>(p.out) + static_cast<int64_t>(sq.first + row / p.group) * p.out_stride +
                            (static_cast<int64_t>(head) * p.group + row % p.group) * HD + d0,
                        x);
      } else {
        store_any<float, V>(rec + rr * HD + d0, x);
        if (lane == 0 && rp % PARTS == 0) rec[RG * HD + 2 * rr] = top, rec[RG * HD + 2 * rr + 1] = sum;
      }
    }
    // the next run's tiles go where the sums lay; s_m, s_l and q are written again
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
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
  const FewSeq fs = few_seq<HD, NT>(p, seq);
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
    const FewSeq f = few_seq<HD, NT>(p, s);
    const int64_t v = f.cost() * f.groups * kvh;
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
  const int64_t lo = before + (rg * kvh + head) * fs.cost(), hi = lo + fs.cost();
  const int64_t ctas = few_ctas(total, grid_ctas);
  // CTA i holds [total * i / ctas, total * (i + 1) / ctas): the one of granule x
  auto owner = [&](int64_t x) {
    int64_t i = x * ctas / total;
    while (total * (i + 1) / ctas <= x) ++i;
    while (total * i / ctas > x) --i;
    return static_cast<int>(i);
  };
  const int c0 = owner(lo + few_unit_cost(HD)), n = owner(hi - 1) - c0 + 1;
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
