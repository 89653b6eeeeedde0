// kvq8_many.cuh -- attention of many rows per sequence (prompts, prefill
// chunks) over the paged 8-bit cache, on the 5th-generation tensor cores.
//
// Two kernels.  kvq8_gather_kernel unpacks each sequence's pages once per call
// into the workspace: K as half codes [head][key][d], V transposed, [head][d]
// [key] (so both products take K-major operands), keys padded to whole tiles
// of 128, with the scales of every 16 keys; its last CTA lays out the work.
// Per key, head and dimension that is 2 bytes read and 4 written, against 4
// flops for every query row: little for the 128 and more rows it serves.
//
// kvq8_many_kernel, one CTA per SM, works through an equal run of (unit, 128
// keys) granules (a unit: 128 query rows of one KV head, row = token * group +
// query head, so the heads of a group share every K and V tile), like the
// few-row kernel; units that cross CTAs leave records for kvq8_many_merge.
//   warp 8      streams K and V tiles by tensor-map TMA (128-byte swizzle, no
//               multicast) through a ring of up to 32 KB stages;
//   warp 9      issues the MMAs: S(j) = Q K^T into one of two TMEM buffers
//               (M = 128, N = 128), then O += P(j-1) V (N = head_dim) with P
//               read from TMEM: the softmax of one tile runs under the
//               products of its neighbours;
//   warps 0-7   softmax: a thread has 64 of a row's 128 scores, p =
//               2^(s - m), and writes p * v_scale back over S as halves.  m
//               moves only when a row's maximum grows by more than 2^8, so O
//               is rarely rescaled.
// Numerics as in the few-row kernel: codes are exact in half; half rows use q
// as given and p as one half (2^7 above the largest v_scale of the run: room
// for the 2^8); fp32 rows use q and p as high + low halves, twice the MMAs.
// TMEM: O in columns 0 .. head_dim - 1, S in 256.. and 384..
//
// The tensor core's fp32 sums are cut toward zero: a step (16 keys) loses up
// to 2^-22 of the sum where V are all alike, some 2e-8 where their signs are
// random.  For half rows O is summed in TMEM all the same, over at most 256
// tiles, where that stays under half's 2^-11, and joined with rounding from
// there on (two sequences of 2048 rows after 131072 keys of 64 dimensions:
// error 2.6e-3 -> 1.1e-3 where values are alike, 7.1e-4 -> 5.3e-4 where not).
// Of fp32 rows a tile's products are summed from zero, low halves first, and
// the softmax threads add them to O in their registers with rounding (l takes
// along what its additions round off): two warpgroups hold half a row of O
// each, 128 registers a thread at 256 dimensions, which the helpers' warpgroup
// gives up (setmaxnreg).  Error against 64 bits after 6144 keys: 0.35e-6 of a
// random result, 1.9e-6 at most where one key holds the weight and V are alike.
// (Summed in TMEM and moved into sums in memory every 8 tiles: 1.4e-6 with a
// correction for random data, 13e-6 for the other; prompts of up to 3001
// tokens 307 us where this takes 278.  Halves by this form: 258 us instead of
// 228 for the chunk below.)
//
// Bound by the tensor pipe where runs are long (1024 half rows of 8 heads of
// 256 after 32768 keys: 228-252 us by the machine, up to 1190 TFLOP/s; fp32 391 us),
// by what a unit costs besides its tiles where they are short (prompts
// of up to 3001 tokens: halves 181 us, fp32 278 us).  Two turns of softmax
// warps on alternate tiles instead of two halves of each took 280 us for the
// former, asking for the next stage before a tile's products 252.
//
// Every wait is bounded; one that gives up raises *err, and all roles still
// walk their loops to the end (without touching TMEM) so that no barrier is
// left short of threads.
#pragma once

#include "gemm_tc.cuh"
#include "kvq8_few.cuh"

namespace kib {

constexpr int kManyRows = 128;   // query rows of a unit
constexpr int kManyKeys = 128;   // keys of a granule
constexpr int kManySoft = 256;   // softmax threads

// A unit costs about as much as this many granules besides its own (q in, the
// pipeline filled and drained, O out), so runs are cut by granules plus this:
// without it the CTA at the start of a prompt, where a unit sees one to three
// tiles of keys, takes 26 units where others take 3.  Five prompts of up to
// 3001 tokens, head_dim 256, 8 query heads, halves / fp32: 321 / 507 us with a
// cost of 1, 261 / 412 with 2, 208 / 325 with 4, 178 / 273 with 6, 197 / 320
// with 16 (head_dim 128: 6 is best too).
constexpr int kManyUnitCost = 6;

// Tiles of a half rows' run at most: longer ones are cut, and joined as if by
// another CTA, in this one's record.
constexpr int kManyRun = 256;

struct Kvq8ManyParams {
  Kvq8AttnParams a;
  int tot_pad;      // padded keys that the workspace holds
  int max_units;
  __half* k16;      // [kv_heads][tot_pad][head_dim]
  __half* v16;      // [kv_heads][head_dim][tot_pad]
  float2* scales;   // [kv_heads][tot_pad / 16]: k and v scale; v < 0: an absent page
  int* seq_off;     // [sequences + 1] first padded key
  int4* units;      // [max_units] sequence, row tile, head, granules
  int64_t* cum;     // [max_units + 1] running cost; cum[count[0]] is the total
  int* cta_unit;    // [ctas] unit at which a CTA begins
  int4* split;      // [ctas] units that cross CTAs: unit, first CTA, CTAs, whether its first record is a CTA's second
  int* count;       // [2] units, split units
  int ctas;
  int* err;
};

// Rows and visible keys of a sequence that this path takes (rows 0: not its).
struct ManySeq {
  int n, tiles, span, pad;
};
KIB_DEV ManySeq many_seq(const Kvq8AttnParams& p, int s) {
  const Kvq8Seq q = kvq8_seq(p.b, s);
  ManySeq m{0, 0, 0, 0};
  const int64_t rows = static_cast<int64_t>(q.n) * p.group;
  if (q.n > 0 && rows > p.few_limit) {
    m.n = q.n;
    m.tiles = static_cast<int>((rows + kManyRows - 1) / kManyRows);
    m.span = max(0, min(q.length, p.b.max_length));
    m.pad = max(1, (m.span + kManyKeys - 1) / kManyKeys) * kManyKeys;
  }
  return m;
}

// Exclusive scan of v over the block's threads; *total gets the sum.
KIB_DEV int64_t many_scan(int64_t v, int64_t* s, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) s[warp] = inc;
  __syncthreads();
  int64_t base = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) base += s[w];
    all += s[w];
  }
  *total = all;
  return base + inc - v;
}

constexpr int kGatherThreads = 256;

// Grid (tot_pad / 128 + 1, kv_heads): a tile of 128 keys of one head each;
// the last x lays out the work (head 0 only).
template <int HD>
__global__ void __launch_bounds__(kGatherThreads) kvq8_gather_kernel(const __grid_constant__ Kvq8ManyParams p) {
  constexpr int LD = HD + 4;  // bytes of a V row in shared memory
  // first the offsets of the sequences, then the tile's V codes
  constexpr int OFF = (kFewMaxSeqs + 1) * 4, VB = kManyKeys * LD;
  __shared__ __align__(16) uint8_t s_raw[OFF > VB ? OFF : VB];
  int* s_off = reinterpret_cast<int*>(s_raw);
  uint8_t* s_v = s_raw;
  __shared__ int64_t s_scan[kGatherThreads / 32];  // 64 bits: lengths and row starts may be wrong, their sums too
  const int tid = threadIdx.x, S = p.a.b.sequences, kvh = p.a.c.kv_heads, head = blockIdx.y;
  const bool plan = blockIdx.x + 1 == gridDim.x;
  if (plan && head) return;

  // first padded keys; in the planning CTA then first units
  int64_t base = 0;
  for (int s0 = 0; s0 < S; s0 += kGatherThreads) {
    const int s = s0 + tid;
    const int64_t v = s < S ? many_seq(p.a, s).pad : 0;
    int64_t all;
    const int64_t x = base + many_scan(v, s_scan, &all);
    // a sequence that the workspace has no room for keeps no keys
    if (s < S) s_off[s] = static_cast<int>(min(x, static_cast<int64_t>(p.tot_pad)));
    base += all;
  }
  if (tid == 0) s_off[S] = static_cast<int>(min(base, static_cast<int64_t>(p.tot_pad)));
  __syncthreads();

  if (plan) {
    for (int s = tid; s <= S; s += kGatherThreads) p.seq_off[s] = s_off[s];
    __syncthreads();
    int64_t all_units = 0;
    for (int s0 = 0; s0 < S; s0 += kGatherThreads) {
      const int s = s0 + tid;
      const int64_t v = s < S ? static_cast<int64_t>(many_seq(p.a, s).tiles) * kvh : 0;
      int64_t all;
      const int64_t x = all_units + many_scan(v, s_scan, &all);
      if (s < S) s_off[s] = static_cast<int>(min(x, static_cast<int64_t>(p.max_units)));
      all_units += all;
    }
    const int units = static_cast<int>(min(all_units, static_cast<int64_t>(p.max_units)));
    if (tid == 0) s_off[S] = units, p.count[0] = units, p.count[1] = 0;
    __syncthreads();
    int64_t total = 0;
    for (int u0 = 0; u0 < units; u0 += kGatherThreads) {
      const int u = u0 + tid;
      int64_t v = 0;
      if (u < units) {
        int lo = 0, hi = S;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_off[mid] <= u) lo = mid;
          else hi = mid;
        }
        while (lo + 1 < S && s_off[lo + 1] <= u) ++lo;  // past sequences without units
        const ManySeq m = many_seq(p.a, lo);
        const Kvq8Seq q = kvq8_seq(p.a.b, lo);
        const int tile = (u - s_off[lo]) / kvh, h = (u - s_off[lo]) % kvh;
        const int64_t last = min(static_cast<int64_t>(tile + 1) * kManyRows, static_cast<int64_t>(m.n) * p.a.group) - 1;
        const int room = p.tot_pad - p.seq_off[lo];
        const int end = min(min(m.span, room), q.length - q.n + static_cast<int>(last / p.a.group) + 1);
        const int g = max(1, (end + kManyKeys - 1) / kManyKeys);
        p.units[u] = make_int4(lo, tile, h, g);
        v = g + kManyUnitCost;
      }
      int64_t all;
      const int64_t x = total + many_scan(v, s_scan, &all);
      if (u < units) p.cum[u] = x;
      total += all;
    }
    if (tid == 0) p.cum[units] = total;
    __syncthreads();
    const int64_t ctas = few_ctas(total, p.ctas);
    for (int u = tid; u < units; u += kGatherThreads) {
      const int64_t c0 = p.cum[u], c1 = p.cum[u + 1];
      for (int64_t i = (c0 * ctas + total - 1) / total; i < ctas && total * i / ctas < c1; ++i)
        if (total * i / ctas >= c0) p.cta_unit[i] = u;
      // CTA i holds [total * i / ctas, total * (i + 1) / ctas): the one of position x
      auto owner = [&](int64_t x) {
        int64_t i = x * ctas / total;
        while (total * (i + 1) / ctas <= x) ++i;
        while (total * i / ctas > x) --i;
        return static_cast<int>(i);
      };
      const int a = owner(c0 + kManyUnitCost), n = owner(c1 - 1) - a + 1;
      if (n > 1) p.split[atomicAdd(p.count + 1, 1)] = make_int4(u, a, n, total * a / ctas < c0 ? 1 : 0);
    }
    return;
  }

  const int at = blockIdx.x * kManyKeys;  // padded key of this tile
  if (at >= s_off[S]) return;
  int seq;
  {
    int lo = 0, hi = S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_off[mid] <= at) lo = mid;
      else hi = mid;
    }
    seq = lo;
    while (seq + 1 < S && s_off[seq + 1] <= at) ++seq;
  }
  const ManySeq m = many_seq(p.a, seq);
  const int key0 = at - s_off[seq];
  __syncthreads();
  const Kvq8Cache& c = p.a.c;
  constexpr int CH = HD / 16;  // 16-byte chunks of a row
  for (int i = tid; i < kManyKeys * CH; i += kGatherThreads) {
    const int r = i / CH, ch = i % CH, key = key0 + r;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    const int page = key < m.span ? kvq8_page(c, p.a.b, seq, key >> c.page_shift) : -1;
    if (page >= 0) {
      const int64_t off = page * c.page_stride + head * c.head_stride + (key & (c.page_tokens - 1)) * c.token_stride + 16 * ch;
      k = ldg_stream(c.k + off);
      v = ldg_stream(c.v + off);
    }
    const uint32_t w[4] = {k.x ^ 0x80808080u, k.y ^ 0x80808080u, k.z ^ 0x80808080u, k.w ^ 0x80808080u};
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[2 * j] = codes_to_half2(w[j], 0x4140u), h[2 * j + 1] = codes_to_half2(w[j], 0x4342u);
    uint4* dst = reinterpret_cast<uint4*>(p.k16 + (static_cast<int64_t>(head) * p.tot_pad + at + r) * HD + 16 * ch);
    dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
    dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
    uint32_t* sv = reinterpret_cast<uint32_t*>(s_v + r * LD + 16 * ch);
    sv[0] = v.x, sv[1] = v.y, sv[2] = v.z, sv[3] = v.w;
  }
  if (tid < kManyKeys / 16) {
    const int key = key0 + 16 * tid;
    const int page = key < m.span ? kvq8_page(c, p.a.b, seq, key >> c.page_shift) : -1;
    float2 s = make_float2(0.0f, -1.0f);
    if (page >= 0) s = make_float2(c.k_scale[static_cast<int64_t>(page) * kvh + head], c.v_scale[static_cast<int64_t>(page) * kvh + head]);
    p.scales[(static_cast<int64_t>(head) * p.tot_pad + at) / 16 + tid] = s;
  }
  __syncthreads();
  // 8 keys x 4 dimensions a step: byte permutes turn 8 words into 4 rows of 8 halves
  for (int i = tid; i < (HD / 4) * (kManyKeys / 8); i += kGatherThreads) {
    const int oct = (i & 1) + 2 * (i / (2 * (HD / 4))), quad = (i >> 1) % (HD / 4);
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const uint32_t*>(s_v + (8 * oct + j) * LD + 4 * quad);
    uint32_t h[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = prmt(w[2 * j], w[2 * j + 1], 0x5140u) ^ 0x80808080u, hi = prmt(w[2 * j], w[2 * j + 1], 0x7362u) ^ 0x80808080u;
      h[0][j] = codes_to_half2(lo, 0x4140u), h[1][j] = codes_to_half2(lo, 0x4342u);
      h[2][j] = codes_to_half2(hi, 0x4140u), h[3][j] = codes_to_half2(hi, 0x4342u);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d)
      *reinterpret_cast<uint4*>(p.v16 + (static_cast<int64_t>(head) * HD + 4 * quad + d) * p.tot_pad + at + 8 * oct) =
          make_uint4(h[d][0], h[d][1], h[d][2], h[d][3]);
  }
}

// --------------------------------------------------------------- main kernel

KIB_DEV void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// N columns of this thread's lane; the registers are complete when it returns.
KIB_DEV void tmem_ld(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, "
      "%38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, "
      "%56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
      "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
      "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
      "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
      "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
      "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
KIB_DEV void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
      "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
KIB_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
KIB_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
KIB_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp, the same each time.  The whole warp walks the
// producing and the issuing loop, so the descriptors stay in uniform registers.
KIB_DEV bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// Barrier of the softmax threads that also tells whether any of them said yes.
KIB_DEV bool soft_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}

struct ManyShared {
  uint64_t full[8], empty[8], s_full[2], p_full[2], o_done[2], q_full;
  float qs[kManyRows];        // what takes a row's scores back from its power of two, times scale_log2
  float x[2][2][kManyRows];   // row maxima of the two halves, by tile parity
  float red[8];
  uint32_t tmem;
};

// TMEM instructions need the whole warp: one lane's failed wait is everyone's.
KIB_DEV bool warp_ok(bool ok) { return __all_sync(0xffffffffu, ok) != 0; }

// Of the 384 threads that fp32 rows are launched with, registers move from the
// warpgroup of the helpers to the two that hold O: 168 each at launch, so the
// shares may come to 384 * 168 together.
constexpr int kManyHelperRegs = 64, kManySoftRegs = 216;
static_assert(128 * kManyHelperRegs + 256 * kManySoftRegs <= 384 * 168, "more registers than the launch has");

template <int HD, int PL>
struct ManyShape {
  static constexpr int kTile = 128 * HD * 2;                      // bytes of a K or a V tile
  static constexpr int kStage = kTile < 32768 ? kTile : 32768;
  static constexpr int kPer = kTile / kStage;                     // stages of a tile
  static constexpr int kQ = PL * kManyRows * HD * 2;
  static constexpr int kStages = HD == 256 ? (PL == 2 ? 3 : 5) : (HD == 128 ? (PL == 2 ? 5 : 6) : 8);
  static constexpr bool kHeld = PL == 2;                          // O in the softmax threads' registers
  static constexpr int kThreads = kManySoft + (kHeld ? 128 : 64);
  static constexpr int kPartial = kManyRows * (HD + 2);           // floats of a record
  static constexpr size_t kSmem = static_cast<size_t>(kQ) + kStages * kStage + sizeof(ManyShared);
};

template <int HD, int PL>
__global__ void __launch_bounds__(ManyShape<HD, PL>::kThreads, 1)
    kvq8_many_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ Kvq8ManyParams p) {
  using T = typename std::conditional<PL == 2, float, __half>::type;
  using Sh = ManyShape<HD, PL>;
  // q [PL][HD / 64][128 rows][128 bytes], swizzled; stages; the rest.  All of
  // it dynamic: the first byte is then 1024-byte aligned, as the swizzle needs
  extern __shared__ __align__(1024) uint8_t many_raw[];
  uint8_t* s_q = many_raw;
  uint8_t* s_st = many_raw + Sh::kQ;
  ManyShared& sh = *reinterpret_cast<ManyShared*>(s_st + Sh::kStages * Sh::kStage);
  uint64_t *full = sh.full, *empty = sh.empty, *s_full = sh.s_full, *p_full = sh.p_full;
  // like the S buffers, the products' barriers alternate: at the end of a run two of them may still be running
  uint64_t *o_done = sh.o_done, &q_full = sh.q_full;
  float* s_qs = sh.qs;
  float* s_red = sh.red;
  if (smem_u32(many_raw) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, 3);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  const int64_t total = p.cum[p.count[0]];
  const int64_t ctas = few_ctas(total, p.ctas);
  if (blockIdx.x >= ctas) return;
  const int64_t first = total * blockIdx.x / ctas, stop = total * (blockIdx.x + 1) / ctas;
  const int unit0 = p.cta_unit[blockIdx.x];

  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&s_full[b], 1), mbar_init(&p_full[b], 8), mbar_init(&o_done[b], 1);
    mbar_init(&q_full, 8);
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);

  // every role walks the same runs: granules [g0, g1) of a unit
  struct Run {
    int seq, tile, head, g0, g1;
    bool whole;        // the unit is all this CTA's
    bool later, last;  // there is a run of the unit before this one here, this is its last
    bool done;         // the unit ends with this run
    int slot;          // its record
    int64_t next;
  };
  auto run_at = [&](int unit, int64_t at) {
    const int4 u = p.units[unit];
    const int64_t start = p.cum[unit], c0 = start + kManyUnitCost, c1 = c0 + u.w, mine = min(c1, stop);
    Run r{u.x, u.y, u.z};
    r.next = Sh::kHeld ? mine : min(mine, max(at, c0) + kManyRun);
    r.g0 = static_cast<int>(max(at - c0, static_cast<int64_t>(0)));
    r.g1 = static_cast<int>(max(r.next - c0, static_cast<int64_t>(0)));
    r.whole = first <= c0 && c1 <= stop;
    r.later = at > max(first, start);
    r.last = r.next == mine;
    r.done = r.next == c1;
    r.slot = first >= start ? 0 : 1;
    return r;
  };

  if (warp >= 8) {
    if constexpr (Sh::kHeld) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyHelperRegs));
    if (warp == 8) {
      if (elect_one()) tma_prefetch_desc(&kmap), tma_prefetch_desc(&vmap);
      uint32_t it = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, bool is_k, int head, int key) {
        // K: 128 keys x 64 dimensions a box; V: 64 keys x HD dimensions a box
        constexpr int kBox = 16384, vBox = HD * 128;
#pragma unroll 1
        for (int i = 0; i < Sh::kPer && ok; ++i, ++it) {
          const int s = static_cast<int>(it % Sh::kStages);
          ok = warp_ok(tc_wait(&empty[s], ((it / Sh::kStages) & 1) ^ 1, p.err));
          if (!ok) break;
          uint8_t* dst = s_st + s * Sh::kStage;
          if (!elect_one()) continue;
          mbar_arrive_expect_tx(&full[s], Sh::kStage);
          if (is_k) {
#pragma unroll
            for (int b = 0; b < Sh::kStage / kBox; ++b)
              tma_load_2d(dst + b * kBox, map, (i * (Sh::kStage / kBox) + b) * 64, head * p.tot_pad + key, &full[s]);
          } else {
#pragma unroll
            for (int b = 0; b < Sh::kStage / vBox; ++b)
              tma_load_2d(dst + b * vBox, map, key + (i * (Sh::kStage / vBox) + b) * 64, head * HD, &full[s]);
          }
        }
      };
      int unit = unit0;
      for (int64_t at = first; at < stop && ok;) {
        const Run r = run_at(unit, at);
        at = r.next;
        unit += r.done;
        if (r.g0 == r.g1) continue;
        const int off = p.seq_off[r.seq];
        for (int j = r.g0; j < r.g1 && ok; ++j) {
          load(&kmap, true, r.head, off + j * kManyKeys);
          if (j > r.g0) load(&vmap, false, r.head, off + (j - 1) * kManyKeys);
        }
        if (ok) load(&vmap, false, r.head, off + (r.g1 - 1) * kManyKeys);
      }
    } else if (warp == 9) {
      constexpr uint32_t idesc_s = umma_idesc_f16(kManyKeys), idesc_o = umma_idesc_f16(HD);
      uint32_t it = 0, jg = 0, piece = 0;
      bool ok = true;
      // a descriptor's start address counts 16 bytes, so steps within the operands are additions
      const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), st_desc = umma_desc_sw128(smem_u32(s_st));
      auto scores = [&](uint32_t jj) {
        const uint32_t d = tmem + 256 + 128 * (jj & 1);
        // q's low halves first: the tensor core's sums lose up to their last
        // bits toward zero at every step, least while they are small
#pragma unroll 1
        for (int pl = PL - 1; pl >= 0 && ok; --pl) {
#pragma unroll 1
          for (int i = 0; i < Sh::kPer && ok; ++i) {
            const int s = static_cast<int>((it + i) % Sh::kStages);
            if (pl == PL - 1) {
              ok = warp_ok(tc_wait(&full[s], ((it + i) / Sh::kStages) & 1, p.err));
              if (!ok) break;
              tc_fence_after();
            }
            constexpr int STEPS = HD / 16 / Sh::kPer;
            const uint64_t b0 = st_desc + static_cast<uint64_t>(s * (Sh::kStage / 16)),
                           a0 = q_desc + static_cast<uint64_t>(i * (STEPS / 4) * 1024 + pl * (kManyRows * HD * 2 / 16));
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < STEPS; ++k)
                umma_f16(d, a0 + (k / 4) * 1024 + 2 * (k % 4), b0 + (k / 4) * 1024 + 2 * (k % 4), idesc_s,
                         k != 0 ? 1u : (i != 0 || pl != PL - 1 ? 1u : 0u));
              if (pl == 0) umma_commit(&empty[s]);
              if (pl == 0 && i + 1 == Sh::kPer) umma_commit(&s_full[jj & 1]);
            }
            __syncwarp();
          }
        }
        it += Sh::kPer;
      };
      auto outputs = [&](uint32_t jj, bool begin) {
        ok = warp_ok(ok && tc_wait(&p_full[jj & 1], (jj >> 1) & 1, p.err));
        tc_fence_after();
        const uint32_t a = tmem + 256 + 128 * (jj & 1);
        // fp32 rows: every tile from zero, p's low halves first as q's above
#pragma unroll 1
        for (int pl = PL - 1; pl >= 0 && ok; --pl) {
#pragma unroll 1
          for (int i = 0; i < Sh::kPer && ok; ++i) {
            const int s = static_cast<int>((it + i) % Sh::kStages);
            if (pl == PL - 1) {
              ok = warp_ok(tc_wait(&full[s], ((it + i) / Sh::kStages) & 1, p.err));
              if (!ok) break;
              tc_fence_after();
            }
            constexpr int STEPS = kManyKeys / 16 / Sh::kPer;
            const uint64_t b0 = st_desc + static_cast<uint64_t>(s * (Sh::kStage / 16));
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < STEPS; ++k) {
                const int ks = i * STEPS + k;  // 16 keys
                umma_f16_ts(tmem, Sh::kHeld ? a + 32 * (ks / 2) + 8 * (ks % 2) + 16 * pl : a + 8 * ks, b0 + (k / 4) * (HD * 8) + 2 * (k % 4),
                            idesc_o, k != 0 || i != 0 || pl != PL - 1 ? 1u : (Sh::kHeld || begin ? 0u : 1u));
              }
              if (pl == 0) umma_commit(&empty[s]);
              if (pl == 0 && i + 1 == Sh::kPer) umma_commit(&o_done[jj & 1]);
            }
            __syncwarp();
          }
        }
        it += Sh::kPer;
      };
      int unit = unit0;
      for (int64_t at = first; at < stop && ok;) {
        const Run r = run_at(unit, at);
        at = r.next;
        unit += r.done;
        if (r.g0 == r.g1) continue;
        ok = warp_ok(tc_wait(&q_full, piece++ & 1, p.err));
        tc_fence_after();
        const int n = r.g1 - r.g0;
        for (int j = 0; j < n && ok; ++j) {
          scores(jg + j);
          if (j > 0 && ok) outputs(jg + j - 1, j == 1);
        }
        if (ok) outputs(jg + n - 1, n == 1);
        jg += n;
      }
    }
  } else {
    if constexpr (Sh::kHeld) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManySoftRegs));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;  // columns 64 half .. of TMEM lane `row`
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t jg = 0;
    bool ok = true;
    int unit = unit0;
    for (int64_t at = first; at < stop;) {
      const Run r = run_at(unit, at);
      at = r.next;
      unit += r.done;
      if (r.g0 == r.g1) continue;
      const Kvq8Seq sq = kvq8_seq(p.a.b, r.seq);
      const ManySeq ms = many_seq(p.a, r.seq);
      const int off = p.seq_off[r.seq];
      const int nrows = sq.n * p.a.group, row0 = r.tile * kManyRows;
      const int live = min(kManyRows, nrows - row0);
      const int start = sq.length - sq.n;
      // the workspace may hold fewer keys than the sequence has
      const int span = min(ms.span, p.tot_pad - off);
      auto row_end = [&](int i) { return i < live ? min(span, start + (row0 + i) / p.a.group + 1) : 0; };
      const float2* scales = p.scales + (static_cast<int64_t>(r.head) * p.tot_pad + off) / 16;

      // q rows to shared memory as halves, in the swizzled layout of the MMA;
      // eight of a warp's rows asked for before the first is used (one after
      // the other their latencies add up to 15 us a unit)
      constexpr int V = HD / 32;
#pragma unroll 1
      for (int i0 = warp; i0 < kManyRows; i0 += 64) {
        float xs[8][V];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int rr = row0 + min(i0 + 8 * e, live - 1);
          load_vec<T, V>(static_cast<const T*>(p.a.q) + static_cast<int64_t>(sq.first + rr / p.a.group) * p.a.q_stride +
                             (static_cast<int64_t>(r.head) * p.a.group + rr % p.a.group) * HD + lane * V,
                         xs[e]);
        }
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) {
          const int i = i0 + 8 * i8;
          float (&x)[V] = xs[i8];
          if (i >= live) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = 0.0f;
          }
          // a negative softmax scale goes into q's sign
          if (p.a.scale_log2 < 0.0f) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = -x[e];
          }
          float back = 1.0f;
          if constexpr (PL == 2) {
            float big = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) big = fmaxf(big, fabsf(x[e]));
            big = warp_max(big);
            const int ex = static_cast<int>(__float_as_uint(big) >> 23);
            if (ex > 20 && ex < 255) {
              const int k = min(max(140 - ex, -100), 100);
              const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
              back = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
              for (int e = 0; e < V; ++e) x[e] *= up;
            }
          }
          uint32_t hi[V / 2], lo[V / 2];
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            hi[e / 2] = pack_half2(x[e], x[e + 1]);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[e / 2]));
            lo[e / 2] = pack_half2(x[e] - f.x, x[e + 1] - f.y);
          }
          const int byte = lane * V * 2, slab = byte / 128, ch = (byte % 128) / 16;
          uint8_t* dst = s_q + slab * 16384 + i * 128 + ((ch ^ (i & 7)) * 16) + byte % 16;
#pragma unroll
          for (int e = 0; e < V / 2; ++e) {
            reinterpret_cast<uint32_t*>(dst)[e] = hi[e];
            if constexpr (PL == 2) reinterpret_cast<uint32_t*>(dst + kManyRows * HD * 2)[e] = lo[e];
          }
          if (lane == 0) s_qs[i] = back * fabsf(p.a.scale_log2);
        }
      }
      // the run's largest v_scale
      float vmax = 0.0f;
      for (int i = r.g0 * 8 + threadIdx.x; i < r.g1 * 8; i += kManySoft) vmax = fmaxf(vmax, __ldg(scales + i).y);
      vmax = warp_max(vmax);
      if (lane == 0) s_red[warp] = vmax;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      soft_any(false);
      if (lane == 0) mbar_arrive(&q_full);
#pragma unroll
      for (int w = 0; w < 8; ++w) vmax = fmaxf(vmax, s_red[w]);
      const int ve = min(max(static_cast<int>(__float_as_uint(vmax) >> 23), 20), 254);
      const float vup = __uint_as_float(static_cast<uint32_t>(min(260 - ve, 254)) << 23);  // 2^7 / 2^(ve - 126)
      const float qs = s_qs[row];
      const int end = row_end(row);
      const int all_see = row_end(0);  // keys below it are seen by every row (of the dead ones nothing is kept)

      float m = -INFINITY, l = 0.0f;
      // m is a rounded product: where a score's last bit may be 2^-4 and above, s * kc is rounded by itself too
      auto is_large = [](float x) { return fabsf(x) > 0x1p20f && x != -INFINITY; };
      bool large = false;
      const int n = r.g1 - r.g0;
      float2 sc[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) sc[g] = __ldg(scales + r.g0 * 8 + half * 4 + g);
      // O of the product before last or last: complete when S of the tile after it is, or with this wait
      auto wait_o = [&](uint32_t jj) {
        ok = warp_ok(ok && tc_wait(&o_done[jj & 1], (jj >> 1) & 1, p.err));
        tc_fence_after();
      };
      [[maybe_unused]] float held[Sh::kHeld ? HD / 2 : 1], lc = 0.0f;  // O; what the last addition to l rounded off
      if constexpr (Sh::kHeld) {
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) held[i] = 0.0f;
      }
      // O += f * the sum of one tile
      auto add_tile = [&](float f) {
        if constexpr (Sh::kHeld) {
#pragma unroll
          for (int c0 = 0; c0 < HD / 2; c0 += 32) {
            uint32_t o[32];
            tmem_ld(tmem + lanes + half * (HD / 2) + c0, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) held[c0 + i] = fmaf(__uint_as_float(o[i]), f, held[c0 + i]);
          }
        }
      };
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const uint32_t jj = jg + j, buf = jj & 1;
        const int key = (r.g0 + j) * kManyKeys + half * 64;
        float kc[4], vc[4];
        bool absent = false;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          kc[g] = sc[g].x * qs;
          vc[g] = sc[g].y * vup;
          absent = absent || sc[g].y < 0.0f;
        }
        // what is masked goes to -infinity; kc is not negative, so a group's largest score is that of its largest s
        const bool edge = key + 64 > all_see || absent;
        if (edge) {
#pragma unroll
          for (int g = 0; g < 4; ++g) kc[g] = fmaxf(kc[g], 1e-38f);  // 0 times -infinity would be NaN
        }
        ok = warp_ok(ok && tc_wait(&s_full[buf], (jj >> 1) & 1, p.err));
        tc_fence_after();
        const uint32_t src = tmem + lanes + 256 + 128 * buf + 64 * half;
        // scores are held 64 at a time, or (next to O) read 32 at a time, for their maximum and again for their weights
        constexpr int CH = Sh::kHeld ? 32 : 64;
        uint32_t s[CH];
        auto load = [&](int c0) {
          if (ok) tmem_ld(src + c0, s);
          if (edge) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
              if (key + c0 + i >= end || sc[(c0 + i) >> 4].y < 0.0f) s[i] = 0xff800000u;
          }
        };
        float top = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += CH) {
          load(c0);
#pragma unroll
          for (int g = 0; g < CH / 16; ++g) {
            float a = __uint_as_float(s[16 * g]), b = __uint_as_float(s[16 * g + 1]);
#pragma unroll
            for (int i = 2; i < 16; i += 4) {
              a = fmaxf(fmaxf(a, __uint_as_float(s[16 * g + i])), i + 2 < 16 ? __uint_as_float(s[16 * g + i + 2]) : a);
              b = fmaxf(fmaxf(b, __uint_as_float(s[16 * g + i + 1])), i + 3 < 16 ? __uint_as_float(s[16 * g + i + 3]) : b);
            }
            top = fmaxf(top, fmaxf(a, b) * kc[c0 / 16 + g]);
          }
        }
        sh.x[buf][half][row] = top;
        // m follows only a growth of more than 2^8: p stays below 2^8, its half below 2^15
        [[maybe_unused]] float last_f = 1.0f;  // for the tile that is not in O yet
        if (soft_any(top > m + 8.0f)) {
          const float mn = fmaxf(m, fmaxf(top, sh.x[buf][half ^ 1][row]));
          const float f = m == -INFINITY ? 0.0f : ex2(m - mn);
          m = mn;
          if constexpr (!Sh::kHeld) large = __any_sync(0xffffffffu, is_large(m));
          l *= f;
          if constexpr (Sh::kHeld) {
            lc *= f;
            last_f = f;
#pragma unroll
            for (int i = 0; i < HD / 2; ++i) held[i] *= f;
          } else if (j > 0) {
            // S(j) was issued after the product before last, so only the last one may still run
            wait_o(jj - 1);
            if (ok) {
#pragma unroll 1
              for (int c0 = 0; c0 < HD / 2; c0 += 32) {
                uint32_t o[32];
                const uint32_t addr = tmem + lanes + half * (HD / 2) + c0;
                tmem_ld(addr, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(addr, o);
              }
              tmem_st_wait();
            }
          }
        }
        const float mm = m == -INFINITY ? 0.0f : m;
        // two scores an instruction: s * kc - m, and p * v_scale
        float2 lp[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 nm = make_float2(-mm, -mm);
        auto round_products = [&](int c0, int n) {
#pragma unroll
          for (int i = 0; i < n; ++i) s[i] = __float_as_uint(__fmul_rn(__uint_as_float(s[i]), kc[(c0 + i) >> 4]));
#pragma unroll
          for (int g = 0; g < n / 16; ++g) kc[c0 / 16 + g] = 1.0f;
        };
        if constexpr (Sh::kHeld) large = is_large(m);
        else if (large) round_products(0, CH);
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          if constexpr (Sh::kHeld) load(c0);
          constexpr int B = CH == 64 ? 1 : 0;
          if (Sh::kHeld && large) round_products(c0, CH);
          uint32_t ph[16], pl[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const int g = (c0 + i) >> 4, at_s = B * c0 + i;
            float2 e = __ffma2_rn(make_float2(__uint_as_float(s[at_s]), __uint_as_float(s[at_s + 1])), make_float2(kc[g], kc[g]), nm);
            e = make_float2(ex2(e.x), ex2(e.y));
            lp[(i >> 1) & 1] = __fadd2_rn(lp[(i >> 1) & 1], e);
            const float2 w = __fmul2_rn(e, make_float2(vc[g], vc[g]));
            ph[i >> 1] = pack_half2(w.x, w.y);
            if constexpr (PL == 2) {
              const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&ph[i >> 1]));
              pl[i >> 1] = pack_half2(w.x - f2.x, w.y - f2.y);
            }
          }
          // halves: 64 columns of the tile's 128 keys; fp32 rows: 32 keys' high and low halves where their scores were
          if (ok) {
            tmem_st16(Sh::kHeld ? src + c0 : tmem + lanes + 256 + 128 * buf + 32 * half + c0 / 2, ph);
            if constexpr (PL == 2) tmem_st16(src + c0 + 16, pl);
          }
        }
        const float lt = (lp[0].x + lp[0].y) + (lp[1].x + lp[1].y);
        if constexpr (Sh::kHeld) {
          const float y = __fsub_rn(lt, lc), t = __fadd_rn(l, y);
          lc = __fsub_rn(__fsub_rn(t, l), y);
          l = t;
        } else {
          l += lt;
        }
        if (j + 1 < n) {
#pragma unroll
          for (int g = 0; g < 4; ++g) sc[g] = __ldg(scales + (r.g0 + j + 1) * 8 + half * 4 + g);
        }
        if (ok) tmem_st_wait();
        if constexpr (Sh::kHeld) {
          // the products of the tile before, while those of this one wait for it
          if (j > 0) {
            wait_o(jj - 1);
            if (ok) add_tile(last_f);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      jg += n;

      // the unit's or the run's end: O / l, or a record
      wait_o(jg - 1);
      if constexpr (Sh::kHeld) {
        if (ok) add_tile(1.0f);
      }
      float* s_l = reinterpret_cast<float*>(s_q);  // q has been read by every product of the run
      s_l[half * kManyRows + row] = l;
      float* rec = p.a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + r.slot) * Sh::kPartial;
      // the unit's run before this one left its m, l and O there
      float2 before = make_float2(-INFINITY, 0.0f);
      if (!Sh::kHeld && r.later && row < live) before = make_float2(rec[kManyRows * HD + 2 * row], rec[kManyRows * HD + 2 * row + 1]);
      soft_any(false);
      l += s_l[(half ^ 1) * kManyRows + row];
      float back = __uint_as_float(static_cast<uint32_t>(max(ve - 6, 1)) << 23);  // 2^(ve - 126) / 2^7
      if (!Sh::kHeld && r.later) {
        const float mn = fmaxf(m, before.x), f = m == -INFINITY ? 0.0f : ex2(m - mn) * back;
        const float more = before.x == -INFINITY ? 0.0f : ex2(before.x - mn);
        l = fmaf(l, m == -INFINITY ? 0.0f : ex2(m - mn), before.y * more);
        m = mn;
        back = 1.0f;
#pragma unroll 1
        for (int c0 = half * (HD / 2); ok && c0 < (half + 1) * (HD / 2); c0 += 32) {
          uint32_t o[32];
          tmem_ld(tmem + lanes + c0, o);
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float z[8] = {};
            if (row < live) load_vec<float, 8>(rec + row * HD + c0 + i, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i + e] = __float_as_uint(fmaf(z[e], more, __uint_as_float(o[i + e]) * f));
          }
          tmem_st32(tmem + lanes + c0, o);
        }
        if (ok) tmem_st_wait();
      }
      const bool out_now = r.whole && r.last;
      const float inv = out_now ? (l > 0.0f ? back / l : (l == 0.0f ? 0.0f : l)) : back;
      const int rr = row0 + row;
      T* out = static_cast<T*>(p.a.out) + static_cast<int64_t>(sq.first + rr / p.a.group) * p.a.out_stride +
               (static_cast<int64_t>(r.head) * p.a.group + rr % p.a.group) * HD;
      auto put = [&](int c0, const float (&x)[8]) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e] * inv;
        if (out_now) store_vec<T, 8>(out + c0, y);
        else store_vec<float, 8>(rec + row * HD + c0, y);
      };
      if constexpr (Sh::kHeld) {
        if (row < live) {
#pragma unroll
          for (int i = 0; i < HD / 2; i += 8) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = held[i + e];
            put(half * (HD / 2) + i, x);
          }
        }
      } else {
#pragma unroll 1
        for (int c0 = half * (HD / 2); c0 < (half + 1) * (HD / 2); c0 += 32) {
          uint32_t o[32];
          if (ok) tmem_ld(tmem + lanes + c0, o);
          if (row < live) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(o[i + e]);
              put(c0 + i, x);
            }
          }
        }
      }
      if (!out_now && row < live && half == 0) {
        rec[kManyRows * HD + 2 * row] = m;
        rec[kManyRows * HD + 2 * row + 1] = l;
      }
      // O is read: the next run may write it (its P arrives after this), q and the shared rows too
      tc_fence_before();
      soft_any(false);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the records of the units that cross CTAs, in CTA order: a CTA per
// such unit and 8 rows, a warp per row.
template <int HD, int PL>
__global__ void __launch_bounds__(256) kvq8_many_merge(const __grid_constant__ Kvq8ManyParams p) {
  using T = typename std::conditional<PL == 2, float, __half>::type;
  constexpr int64_t REC = ManyShape<HD, PL>::kPartial;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 8 + warp;
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= p.count[1]) return;
  const int4 sp = p.split[blockIdx.x], u = p.units[sp.x];
  const Kvq8Seq sq = kvq8_seq(p.a.b, u.x);
  const int rr = u.y * kManyRows + row, n = sp.z;
  if (rr >= sq.n * p.a.group) return;
  const float* rec0 = p.a.partial + static_cast<int64_t>(sp.y) * 2 * REC;
  const float* rec_first = rec0 + (sp.w ? REC : 0);
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, (i ? rec0 + 2 * REC * i : rec_first)[kManyRows * HD + 2 * row]);
  top = warp_max(top);
  constexpr int V = HD / 32;
  float acc[V] = {}, sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* rec = i ? rec0 + 2 * REC * i : rec_first;
    const float2 ml = *reinterpret_cast<const float2*>(rec + kManyRows * HD + 2 * row);
    const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - top);
    sum += f * ml.y;
    float x[V];
    load_vec<float, V>(rec + row * HD + lane * V, x);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] += f * x[e];
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] *= inv;
  store_vec<T, V>(static_cast<T*>(p.a.out) + static_cast<int64_t>(sq.first + rr / p.a.group) * p.a.out_stride +
                      (static_cast<int64_t>(u.z) * p.a.group + rr % p.a.group) * HD + lane * V,
                  acc);
}

}  // namespace kib
