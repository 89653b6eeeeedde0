// sample.cu -- a token per row of logits by temperature, top-k, top-p and
// min-p from a given uniform number.
//
// With M the row's largest logit, e_i = exp((l_i - M) * (1 / T)) and the
// weight w_i = trunc(e_i * 2^40) as an integer: sums of up to 2^23 weights fit
// 64 bits and are exact, so the token does not depend on the order in which
// they are added.  Candidates are ordered by (logit descending, index
// ascending); top-k keeps the first k, top-p those of them whose predecessors
// hold less than trunc(top_p * total), min-p those with e_i >= min_p; the
// first candidate always stays.  The token is the first in index order whose
// running weight exceeds trunc(u * total of the kept).  NaN logits count as
// -infinity.
#include <string>
#include <type_traits>

#include <cooperative_groups.h>

#include "kib_ctx.cuh"
#include "per_device.hpp"

namespace cg = cooperative_groups;

namespace kib {
namespace {

struct SampleParams {
  const float* logits;
  int64_t row_stride;
  int rows, vocab;
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* token;
  float* prob;
};

typedef unsigned long long u64;

// Order-preserving integer of a logit: NaN as -infinity, -0 as 0.
KIB_DEV float clean_logit(float l) { return l == l ? l + 0.0f : -INFINITY; }
KIB_DEV uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct RowScale {
  float top, inv_t;
};
KIB_DEV float logit_weight(float l, const RowScale& r) {
  // infinitely far below the top (with +infinity on top: all but such logits)
  const float d = l == r.top ? 0.0f : __fsub_rn(l, r.top);
  if (d == -INFINITY) return 0.0f;
  const float z = __fmul_rn(d, r.inv_t);
  return expf(z);
}
// trunc(e * 2^40) for e in [0, 1] by shifting the significand (conversions to
// 64-bit integers run at a sixteenth of the rate).
KIB_DEV u64 fixed_weight(float e) {
  const uint32_t b = __float_as_uint(e);
  const int shift = static_cast<int>(b >> 23) - 110;  // exponent - 23 + 40
  const uint32_t m = (b & 0x7fffffu) | 0x800000u;
  if (shift >= 0) return static_cast<u64>(m) << shift;
  return shift > -24 ? m >> -shift : 0u;
}

// A cluster of C CTAs takes one row (C = 1 where rows fill the GPU), each a
// slice of its indices, which it reads two to four times, after the first time
// from L2: its maximum; a histogram over the bits of e where a cut is wanted;
// what is kept, summed in warps' segments of the index order.
//
// top-k hides most of a row before the histogram: k of a CTA's threads' maxima
// are k tokens, so no token below the k-th maximum (found bit by bit with block
// counts) is among the first k.  What is left goes to a list, and everything
// else works on it.
//
// The histogram has kBins bins over the bits of e (32 bins an octave: ordered
// like e, near-uniform in log e, so a vocabulary spreads over hundreds of bins;
// atomics on one word run one after another).  A bin takes two 32-bit shared
// atomics a token, its count and the sum of the 18 low bits that the bin leaves
// open, folded into 64-bit masses every 2^14 tokens, before they can overflow:
// both cuts follow from them.  The tokens of the bin with the boundary are
// listed by a pass that also sums what lies above it, and two histograms of
// nine bits each narrow the bin to one value of e.  Where a cut falls inside a
// group of equal e, the group is ordered by its logits (different logits may
// round to one e), then by index.
//
// The CTAs add up their histograms over distributed shared memory: each adds
// its non-zero bins to share b / (bins / C) of CTA r by remote atomics
// (integers: in any order the same), then everyone gathers the shares and scans
// them redundantly, one cluster barrier a histogram.  Three copies of the small
// histogram's share take turns: a copy is cleared behind the barrier after the
// one it was gathered behind, a barrier before its next use.

// Bound by latency.  A CTA's 1024 threads of 64 registers are all that an SM
// holds: of 223 us for 256 rows with settings of every kind its 39 warp
// instructions for 32 logits issue in 66, loads and barriers stall the rest
// (long scoreboard 5.0, barrier 2.2 issue slots an instruction), and 256 rows are two
// waves.  Where few rows are spread wide it is the barriers and scans (32 rows:
// 12 of 46 us issue; loads 3.6, barriers 3.5).  At 248320
// logits, all rows alike: 256 rows with top-k 50 111 us and with top-p 0.9
// besides 124 (the logits move at HBM's rate in 39), top-p 0.9 alone 272,
// neither 114; 32 rows 26, 33, 46, 21 us; one row 21, 31, 27, 15 us.

constexpr int kClusterMax = 16;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1536;     // 32 an octave: from bin 1281 on e < 2^-40, without weight
constexpr int kBinShift = 18;   // of the bits of e
constexpr int kWeighty = 1281;
constexpr int kFine = 512;      // bins of the histograms on the list
constexpr int kListMax = 8192;
constexpr uint32_t kOneBits = 0x3f800000u;

struct SampleShared {
  uint32_t cnt[kBins], low[kBins];    // this CTA's histogram
  u64 mass[kBins];                    // its share of the cluster's (kBins / C of them)
  uint32_t count[kBins];
  uint32_t fcnt[kFine], flow[kFine];  // the small one, and three copies of its share
  u64 fine[3][kFine];
  u64 scan[kWarps], segment[kWarps];
  uint32_t list[kListMax], list_bits[kListMax];
  u64 total, before, here;
  float top, tops[kWarps];
  int first, bin, index, listed;
  uint32_t kmin, kmax;
};

// Weight of a value of e from its bits, and of a bin from its count and the
// (likewise shifted) sum of the bits below `open`: trunc(2^40 e) shifts the
// significand by an amount that is one for a whole bin.
KIB_DEV int low_shift(uint32_t bits) { return max(0, 110 - static_cast<int>(bits >> 23)); }
KIB_DEV u64 bin_mass(uint32_t top_bits, uint32_t count, uint32_t low) {
  if (!count) return 0;
  const int shift = static_cast<int>(top_bits >> 23) - 110;
  const u64 m = (top_bits & 0x7fffffu) | 0x800000u;
  if (shift >= 0) return (m * count + low) << shift;
  return shift > -24 ? (m >> -shift) * count + low : 0u;
}

// The same 2^40 e in two pieces, 2^22 hi + lo, added to sums: additions that
// round towards zero leave the wanted bits in the significand (hi: 2^5 has an
// ulp of 2^-18; the rest, below 2^-18, then lo: 2^-17 has one of 2^-40).  Up to
// 2^10 values fit 32 bits.
struct SplitSum {
  uint32_t hi = 0, lo = 0;
  KIB_DEV void add(float e) {
    const float a = __fadd_rz(e, 32.0f);
    const float rest = e - (a - 32.0f);  // both exact
    hi += __float_as_uint(a) - 0x42000000u;
    lo += __float_as_uint(__fadd_rz(rest, 0x1p-17f)) - 0x37000000u;
  }
  KIB_DEV u64 value() const { return (static_cast<u64>(hi) << 22) + lo; }
};

template <typename T>
KIB_DEV T* peer(cg::cluster_group& cl, T* p, unsigned rank) {
  return cl.map_shared_rank(p, rank);
}

// Exclusive scan over the block; *total gets the sum.  Every warp scans the
// warps' sums for itself: fewer instructions than a loop, and one barrier less
// than having one warp do it.
template <int THREADS>
KIB_DEV u64 block_scan(u64 v, u64* s, u64* total) {
  constexpr int W = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) s[warp] = inc;
  __syncthreads();
  const u64 w = lane < W ? s[lane] : 0;
  u64 winc = w;
#pragma unroll
  for (int o = 1; o < W; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, winc, o);
    if (lane >= o) winc += n;
  }
  *total = __shfl_sync(0xffffffffu, winc, W - 1);
  return __shfl_sync(0xffffffffu, winc - w, warp) + inc - v;
}

__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t sample_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int row = static_cast<int>(blockIdx.x) / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = p.vocab, quads = (V + 3) / 4;
  const int qa = static_cast<int>(static_cast<int64_t>(quads) * rank / C), qb = static_cast<int>(static_cast<int64_t>(quads) * (rank + 1) / C);
  const int Q = qb - qa;
  auto segment_at = [&](int s) { return qa + static_cast<int>(static_cast<int64_t>(Q) * s / kWarps); };
  const float* x = p.logits + static_cast<int64_t>(row) * p.row_stride;
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const float t = p.temperature ? __ldg(p.temperature + row) : 1.0f;
  const int k = p.top_k ? __ldg(p.top_k + row) : 0;
  const float top_p = p.top_p ? __ldg(p.top_p + row) : 1.0f;
  const float min_p0 = p.min_p ? __ldg(p.min_p + row) : 0.0f;
  const float min_p = min_p0 > 0.0f ? fminf(min_p0, 1.0f) : 0.0f;
  const float u = __ldg(p.uniform + row), inv_t = __fdiv_rn(1.0f, t);

  auto load = [&](int q) -> float4 {
    if (wide && 4 * q + 3 < V) return __ldg(reinterpret_cast<const float4*>(x) + q);
    float4 l;
    l.x = 4 * q < V ? __ldg(x + 4 * q) : -INFINITY;
    l.y = 4 * q + 1 < V ? __ldg(x + 4 * q + 1) : -INFINITY;
    l.z = 4 * q + 2 < V ? __ldg(x + 4 * q + 2) : -INFINITY;
    l.w = 4 * q + 3 < V ? __ldg(x + 4 * q + 3) : -INFINITY;
    return l;
  };
  // four quads, `step` apart, all asked for before the first is used; what(first token, logits) of each
  auto for_four = [&](int q, int step, int end, auto what) {
    float4 l[4];
    if (wide && q + 3 * step < min(end, V / 4)) {
#pragma unroll
      for (int w = 0; w < 4; ++w) l[w] = __ldg(reinterpret_cast<const float4*>(x) + q + w * step);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        l[w] = q + w * step < end ? load(q + w * step) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) what(4 * (q + w * step), l[w]);
  };
  auto max4 = [](float4 l) { return fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)); };  // (of NaN and a number: the number)

  float own_top = -INFINITY;
  for (int q = qa + tid; q < qb; q += 4 * kThreads) for_four(q, kThreads, qb, [&](int, float4 l) { own_top = fmaxf(own_top, max4(l)); });
  own_top += 0.0f;
  float top = warp_max(own_top);
  if (lane == 0) sh.tops[warp] = top;
  if (tid == 0) sh.first = 0x7fffffff, sh.index = 0, sh.listed = 0, sh.bin = kBins - 1, sh.before = 0;
  for (int b = tid; b < kBins; b += kThreads) sh.cnt[b] = sh.low[b] = sh.count[b] = 0, sh.mass[b] = 0;
  if (tid < kFine) sh.fcnt[tid] = sh.flow[tid] = 0, sh.fine[0][tid] = sh.fine[1][tid] = sh.fine[2][tid] = 0;
  __syncthreads();
  top = warp_max(sh.tops[lane]);
  if (C > 1) {
    if (tid == 0) sh.top = top;
    cl.sync();
    top = warp_max(lane < C ? *peer(cl, &sh.top, lane) : -INFINITY);
  }

  if (top == -INFINITY || !(t > 1e-6f)) {
    int best = 0x7fffffff;
    if (top > -INFINITY)
      for (int q = qa + tid; q < qb; q += 4 * kThreads)
        for_four(q, kThreads, qb, [&](int i, float4 l) {
          if (max4(l) == top) best = min(best, i + (l.x == top ? 0 : (l.y == top ? 1 : (l.z == top ? 2 : 3))));
        });
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0 && best != 0x7fffffff) atomicMin(&sh.first, best);
    cl.sync();
    if (rank == 0 && warp == 0) {
      best = __reduce_min_sync(0xffffffffu, lane < C ? *peer(cl, &sh.first, lane) : 0x7fffffff);
      if (lane == 0) {
        p.token[row] = best == 0x7fffffff ? -1 : best;
        if (p.prob) p.prob[row] = best == 0x7fffffff ? 0.0f : 1.0f;
      }
    }
    cl.sync();  // no CTA leaves while another may read its shared memory
    return;
  }
  const RowScale rs{top, inv_t};
  const bool by_k = k > 0 && k < V, by_p = !(top_p >= 1.0f);
  const uint32_t min_bits = __float_as_uint(min_p);
  float least = -INFINITY;  // logits below it are not among the first k
  if (by_k && k <= kThreads) {
    const uint32_t key = order_key(own_top) >> 16;
    uint32_t at = 0;
    for (int bit = 15; bit >= 0; --bit)
      if (__syncthreads_count(key >= (at | 1u << bit)) >= k) at |= 1u << bit;
    at <<= 16;
    const float l = __uint_as_float(at & 0x80000000u ? at ^ 0x80000000u : ~at);
    if (l > -INFINITY) least = l;  // (a key below -infinity's is a NaN's)
  }
  const bool hides = least > -INFINITY;
  // e of four logits; without branches (a NaN gives 0)
  auto weights = [&](float4 l, float (&e)[4]) {
    const float x4[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = fmaxf(expf(__fmul_rn(x4[j] == rs.top ? 0.0f : __fsub_rn(x4[j], rs.top), rs.inv_t)), 0.0f);
  };
  auto logit_key = [&](int i) { return order_key(clean_logit(__ldg(x + i))); };
  auto e_bin = [](uint32_t bits) { return min(static_cast<int>(kOneBits >> kBinShift) - static_cast<int>(bits >> kBinShift), kBins - 1); };
  auto bin_bits = [](int bin) { return ((kOneBits >> kBinShift) - static_cast<uint32_t>(bin)) << kBinShift; };  // its smallest
  // A logit of which, and so of all below, e surely has smaller bits: spares
  // their exponentials.  (e grows with the logit, up to the exponential's own
  // error: 1e-3 leaves more than that, and rounding; -infinity if it does not.)
  auto below = [&](uint32_t bits) {
    if (bits < 0x00800000u) return -INFINITY;
    const float z = logf(__uint_as_float(bits)) - 1e-3f, l = rs.top + z * t;
    return l < rs.top && __fmul_rn(__fsub_rn(l, rs.top), rs.inv_t) < z + 5e-4f ? l : -INFINITY;
  };

  // What is kept: bits of e above cut.bits; of those equal to it, all, or
  // (partial) those with a logit key above cut.key, and with it up to index cut.last.
  struct {
    uint32_t bits, key;
    int last;
    bool partial;
  } cut = {0u, 0u, 0x7fffffff, false};
  auto in_cut = [&](int i, uint32_t b) {
    if (b != cut.bits || !cut.partial) return b >= cut.bits;
    const uint32_t key = logit_key(i);
    return key > cut.key || (key == cut.key && i <= cut.last);
  };

  // Of the values that a thread holds, in scan order over the threads: sets
  // sh.bin, sh.before, sh.here where the running sum acc reaches want.
  auto find = [&](const u64* v, auto per_thread, u64 acc, u64 want) {
    constexpr int PER = decltype(per_thread)::value;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (acc < want && want <= acc + v[e]) sh.bin = tid * PER + e, sh.before = acc, sh.here = v[e];
      acc += v[e];
    }
    __syncthreads();
  };
  // The cluster's sums of the small histogram, scanned for `want`; the bin (in
  // descending order), with what lies before it and in it.
  int turn = 0;
  const int fper = kFine / C, per = kBins / C;
  auto find_fine = [&](bool masses, uint32_t top_bits, int open, u64* before, u64* here, u64 want) -> int {
    const int mine_at = turn;
    turn = turn == 2 ? 0 : turn + 1;
    __syncthreads();
    u64 v = 0;
    if (tid < kFine) {
      const uint32_t count = sh.fcnt[tid];
      v = masses ? bin_mass(top_bits | static_cast<uint32_t>(kFine - 1 - tid) << open, count, sh.flow[tid]) : count;
      sh.fcnt[tid] = sh.flow[tid] = 0;  // for the next
    }
    if (C > 1) {
      const int r = tid / fper, at = tid % fper;
      if (v) atomicAdd(peer(cl, &sh.fine[mine_at][at], r), v);
      cl.sync();
      // the copy before last has been gathered by everyone
      if (tid < fper) sh.fine[turn == 2 ? 0 : turn + 1][tid] = 0;
      v = tid < kFine ? *peer(cl, &sh.fine[mine_at][at], r) : 0;
    }
    if (tid == 0) sh.bin = kFine - 1, sh.before = *before, sh.here = 0;
    u64 total;
    const u64 acc = *before + block_scan<kThreads>(v, sh.scan, &total);
    find(&v, std::integral_constant<int, 1>{}, acc, want);
    *before = sh.before;
    *here = sh.here;
    const int bin = sh.bin;
    __syncthreads();  // sh.bin is written again
    return bin;
  };

  // The tokens with bits of e in [klo, khi], listed, or gone through again and
  // again where there are too many.  The same pass sums the weights of those
  // with bits of at least `from`: `kept_sum` is what of it lies in the warp's segment.
  bool all_listed = false, short_list = false;
  float hidden = -INFINITY;  // logits below it are not counted (where all others are listed)
  u64 kept_sum = 0;
  auto pass = [&](uint32_t klo, uint32_t khi, uint32_t from, auto what) {
    const float skip = below(min(klo, from));
    u64 sum = 0;
    const int s0 = segment_at(warp), s1 = segment_at(warp + 1);
    for (int q = s0 + lane; q < s1; q += 128) {
      SplitSum part;
      for_four(q, 32, s1, [&](int i, float4 l) {
        if (!(max4(l) > skip)) return;  // most quads, where few tokens hold the mass
        float e[4];
        weights(l, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = __float_as_uint(e[j]);
          part.add(b >= from ? e[j] : 0.0f);
          if (b - klo <= khi - klo && b) what(i + j, b);
        }
      });
      sum += part.value();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    kept_sum = sum;
  };
  auto make_list = [&](uint32_t klo, uint32_t khi) {
    if (all_listed) return;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    pass(klo, khi, max(khi + 1, min_bits), [&](int i, uint32_t b) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kListMax) sh.list[at] = static_cast<uint32_t>(i), sh.list_bits[at] = b;
    });
    __syncthreads();
    short_list = sh.listed <= kListMax;
  };
  auto for_list = [&](uint32_t klo, uint32_t khi, auto what) {
    if (short_list) {
      for (int j = tid; j < sh.listed; j += kThreads)
        if (sh.list_bits[j] >= klo && sh.list_bits[j] <= khi) what(static_cast<int>(sh.list[j]), sh.list_bits[j]);
    } else {
      const u64 keep = kept_sum;
      pass(klo, khi, 0xffffffffu, what);
      kept_sum = keep;
    }
  };
  // The block's sum, then the cluster's, of a value of each thread.
  auto cluster_sum = [&](u64 v) -> u64 {
    u64 all;
    block_scan<kThreads>(v, sh.scan, &all);
    if (tid == 0) sh.total = all;
    cl.sync();
    u64 sum = lane < C ? *peer(cl, &sh.total, lane) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };

  // Index at which the running sum, in index order, of weight(i, bits of e)
  // over the tokens with bits of at least `floor` exceeds aim_of(total), in the
  // CTA that holds it (-1 in the others); *owner is that CTA's rank.  `ahead`:
  // what the warp's segment holds besides the listed tokens.  First the CTAs'
  // sums, then the segments', then the block goes through one segment.
  auto locate = [&](uint32_t floor, u64 ahead, auto weight, auto aim_of, int* owner, u64* total) -> int {
    __syncthreads();
    if (lane == 0) sh.segment[warp] = ahead;
    __syncthreads();
    for_list(floor, 0xffffffffu, [&](int i, uint32_t b) {
      const u64 v = weight(i, b);
      if (v) atomicAdd(&sh.segment[(kWarps * (i / 4 - qa + 1) - 1) / Q], v);  // the segment that holds quad i / 4
    });
    __syncthreads();
    u64 inc = sh.segment[lane];
    const u64 own = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const u64 all = __shfl_sync(0xffffffffu, inc, 31);
    u64 base = 0, aim;
    if (C > 1) {
      if (tid == 0) sh.total = all;
      cl.sync();
      const u64 theirs = lane < C ? *peer(cl, &sh.total, lane) : 0;
      u64 sums = theirs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += v;
      }
      *total = __shfl_sync(0xffffffffu, sums, 31);
      aim = aim_of(*total);
      *owner = min(__ffs(__ballot_sync(0xffffffffu, sums > aim)) - 1, C - 1);
      base = __shfl_sync(0xffffffffu, sums - theirs, *owner);
      if (*owner != rank) return -1;
    } else {
      *total = all;
      *owner = 0;
      aim = aim_of(all);
    }
    const int seg = min(static_cast<unsigned>(__ffs(__ballot_sync(0xffffffffu, base + inc > aim)) - 1), kWarps - 1u);
    base += __shfl_sync(0xffffffffu, inc - own, seg);
    const int q0 = segment_at(seg), q1 = segment_at(seg + 1);
    for (int at_q = q0; at_q < q1; at_q += kThreads) {
      const int q = at_q + tid;
      u64 w[4] = {0, 0, 0, 0};
      if (q < q1) {
        const float4 l4 = load(q);
        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
        float e[4];
        weights(l4, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = __float_as_uint(e[j]);
          if (b && b >= floor && l[j] >= hidden) w[j] = weight(4 * q + j, b);
        }
      }
      const u64 mine = (w[0] + w[1]) + (w[2] + w[3]);
      u64 block;
      u64 run = base + block_scan<kThreads>(mine, sh.scan, &block);
      if (run <= aim && aim < run + mine) {
        int at = 4 * q;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          run += w[j];
          at += run <= aim;
        }
        sh.index = at;
      }
      base += block;
      if (base > aim) break;
    }
    __syncthreads();
    return sh.index;
  };

  // Moves the cut into bin `bin`, of whose tokens (that pass the cut so far,
  // for masses) `before` already lies ahead, to where the sum reaches want.
  auto select = [&](bool masses, int bin, u64 before, u64 want) {
    const uint32_t klo = bin_bits(bin), khi = min(klo + ((1u << kBinShift) - 1), kOneBits);
    make_list(klo, khi);
    u64 here = 0;
    const int shift = min(low_shift(klo), 31);
    for_list(klo, khi, [&](int i, uint32_t b) {
      if (masses && !in_cut(i, b)) return;
      const int f = kFine - 1 - static_cast<int>(b >> 9 & 511u);
      atomicAdd(&sh.fcnt[f], 1u);
      // rows of more than 2^23 tokens are refused, so 9 bits of each cannot overflow
      if (masses) atomicAdd(&sh.flow[f], (b & 511u) >> shift);
    });
    const uint32_t mid = klo | static_cast<uint32_t>(kFine - 1 - find_fine(masses, klo, 9, &before, &here, want)) << 9;
    for_list(mid, mid + 511u, [&](int i, uint32_t b) {
      if (!masses || in_cut(i, b)) atomicAdd(&sh.fcnt[kFine - 1 - static_cast<int>(b & 511u)], 1u);
    });
    const uint32_t bits = mid | static_cast<uint32_t>(kFine - 1 - find_fine(masses, mid, 0, &before, &here, want));
    const u64 w = masses ? max(fixed_weight(__uint_as_float(bits)), 1ull) : 1;
    u64 ties = (want - before + w - 1) / w;
    const bool partial = ties < here / w || (masses && cut.partial && bits == cut.bits);
    cut.bits = bits;
    cut.partial = partial;
    if (!partial) return;
    // the first `ties` of the tokens with this e: by logit, then by index
    if (tid == 0) sh.kmin = 0xffffffffu, sh.kmax = 0;
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    for_list(bits, bits, [&](int i, uint32_t) {
      const uint32_t key = logit_key(i);
      lo = min(lo, key), hi = max(hi, key);
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) atomicMin(&sh.kmin, lo), atomicMax(&sh.kmax, hi);
    cl.sync();
    lo = __reduce_min_sync(0xffffffffu, lane < C ? *peer(cl, &sh.kmin, lane) : 0xffffffffu);
    hi = __reduce_max_sync(0xffffffffu, lane < C ? *peer(cl, &sh.kmax, lane) : 0u);
    before = 0;
    for (int level = 0; lo < hi && level < 8; ++level) {  // four at most: 2^32 keys, 2^9 a level
      const int open = max(0, 23 - __clz(hi - lo));
      for_list(bits, bits, [&](int i, uint32_t) {
        const uint32_t key = logit_key(i);
        if (key >= lo && key <= hi) atomicAdd(&sh.fcnt[(hi - key) >> open], 1u);
      });
      const uint32_t top_key = hi - (static_cast<uint32_t>(find_fine(false, 0u, 0, &before, &here, ties)) << open), size = 1u << open;
      lo = top_key - lo >= size - 1 ? top_key - (size - 1) : lo;
      hi = top_key;
    }
    cut.key = lo;
    ties -= before;
    int owner;
    u64 total;
    const int at = locate(
        bits, 0, [&](int i, uint32_t b) -> u64 { return b == bits && logit_key(i) == lo; }, [&](u64) { return ties - 1; }, &owner, &total);
    if (C > 1) {
      if (at >= 0 && tid == 0) sh.index = at;
      cl.sync();
      cut.last = *peer(cl, &sh.index, owner);
      cl.sync();  // sh.index is written again
    } else {
      cut.last = at;
      __syncthreads();
    }
  };

  if (by_k || by_p) {
    // 2^14 logits between two folds; backwards, as the slice's end is what L2 surely still holds
    for (int q0 = qa + (Q - 1) / (4 * kThreads) * (4 * kThreads); q0 >= qa; q0 -= 4 * kThreads) {
      const int q = q0 + tid;
      for_four(q, kThreads, qb, [&](int i, float4 l) {
        if (hides && !(max4(l) >= least)) return;
        const float x4[4] = {l.x, l.y, l.z, l.w};
        float e[4];
        weights(l, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = __float_as_uint(e[j]);
          const int bin = e_bin(b);
          const bool counts = bin < kWeighty && (!hides || x4[j] >= least);
          if (hides && counts) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < kListMax) sh.list[at] = static_cast<uint32_t>(i + j), sh.list_bits[at] = b;
          }
          if (counts) {
            atomicAdd(&sh.cnt[bin], 1u);
            atomicAdd(&sh.low[bin], (b & ((1u << kBinShift) - 1)) >> low_shift(b));
          }
        }
      });
      __syncthreads();
      for (int b = tid; b < kBins; b += kThreads) {
        const uint32_t count = sh.cnt[b];
        if (!count) continue;
        const int r = b / per, at = b - r * per;
        const u64 mass = by_p ? bin_mass(bin_bits(b), count, sh.low[b]) : 0;
        if (C == 1) {
          sh.count[b] += count, sh.mass[b] += mass;
        } else {
          atomicAdd(peer(cl, &sh.count[at], r), count);
          if (mass) atomicAdd(peer(cl, &sh.mass[at], r), mass);
        }
        sh.cnt[b] = sh.low[b] = 0;
      }
      __syncthreads();
    }
    if (hides && sh.listed <= kListMax) all_listed = short_list = true, hidden = least;
    cl.sync();
    // the cluster's bins: two to a thread, in the order of the candidates
    constexpr int PER = (kBins + kThreads - 1) / kThreads;
    u64 v[PER], sum = 0, total;
    int k_bin = kBins;  // bins from it on are cut, but for what stays of its own
    u64 k_mass = 0;
    if (by_k) {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = b < kBins ? *peer(cl, &sh.count[b % per], b / per) : 0;
        sum += v[e];
      }
      const u64 acc = block_scan<kThreads>(sum, sh.scan, &total);
      find(v, std::integral_constant<int, PER>{}, acc, static_cast<u64>(k));
      const int bin = sh.bin;
      const u64 before = sh.before;
      __syncthreads();
      if (bin < kWeighty) {  // else every token with weight is kept
        k_bin = bin;
        select(false, bin, before, static_cast<u64>(k));
        if (by_p) {
          const uint32_t klo = bin_bits(bin), khi = min(klo + ((1u << kBinShift) - 1), kOneBits);
          u64 mine = 0;
          for_list(klo, khi, [&](int i, uint32_t b) { mine += in_cut(i, b) ? fixed_weight(__uint_as_float(b)) : 0; });
          k_mass = cluster_sum(mine);
        }
      }
    }
    if (by_p) {
      sum = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = b < min(k_bin, kBins) ? *peer(cl, &sh.mass[b % per], b / per) : (b == k_bin ? k_mass : 0);
        sum += v[e];
      }
      const u64 acc = block_scan<kThreads>(sum, sh.scan, &total);
      const double limit = static_cast<double>(total) * static_cast<double>(top_p);
      const u64 want = limit > 1.0 ? static_cast<u64>(limit) : 1ull;
      find(v, std::integral_constant<int, PER>{}, acc, want);
      const int bin = sh.bin;
      const u64 before = sh.before;
      __syncthreads();
      select(true, bin, before, want);
    }
  }
  // what is kept: listed, or summed above the list's bin and listed in it
  const uint32_t floor = max(cut.bits, min_bits);
  if (!all_listed && (!short_list || cut.bits == 0)) {
    // no cut was found, or its list is too short: all of it once more
    short_list = false;
    kept_sum = 0;
  }
  auto kept = [&](int i, uint32_t b) -> u64 {
    return b != cut.bits || !cut.partial || in_cut(i, b) ? fixed_weight(__uint_as_float(b)) : 0;
  };
  u64 total;
  int owner;
  u64 ahead = all_listed ? 0 : kept_sum;
  if (!short_list) {
    if (cut.partial) {
      // (a list too short for the group of equals)
      u64 sum = 0;
      pass(floor, 0xffffffffu, 0xffffffffu, [&](int i, uint32_t b) { sum += kept(i, b); });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      ahead = sum;
    } else {
      pass(0xffffffffu, 0xffffffffu, floor, [](int, uint32_t) {});
      ahead = kept_sum;
    }
    __syncthreads();
    if (tid == 0) sh.listed = 0;  // all of it is ahead
    short_list = true;
  }
  const int token = locate(floor, ahead, kept,
                           [&](u64 all) -> u64 {
                             const double f = static_cast<double>(all) * static_cast<double>(u);
                             return f > 0.0 ? min(static_cast<u64>(f), all - 1) : 0;
                           },
                           &owner, &total);
  if (token >= 0 && tid == 0) {
    const float e = logit_weight(clean_logit(__ldg(x + token)), rs);
    p.token[row] = token;
    if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(fixed_weight(e)) / static_cast<double>(total));
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

// CTAs of a row: as many as leave all rows on the GPU at once, with slices of
// 2048 logits at least.  More rows than that take one each: 256 rows with top-k
// 50 and top-p 0.9 124 us by one CTA and 172 by two, with top-p alone 272 and
// 302 (rows with settings of every kind mixed even out better by two: 223 and
// 205).
int cluster_of(const SampleParams& p, int num_sms) {
  int c = 1;
  while (c < kClusterMax && static_cast<int64_t>(p.rows) * c * 2 <= num_sms && p.vocab / (2 * c) >= 2048) c *= 2;
  return c;
}

cudaError_t sample_launch(const SampleParams& p, const kib_ctx* ctx, cudaStream_t st) {
  static PerDevice ready;
  cudaError_t e = cudaSuccess;
  ready.once(ctx->device, [&] {
    e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(SampleShared)));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e == cudaSuccess;
  });
  if (e != cudaSuccess) return e;
  const unsigned c = static_cast<unsigned>(cluster_of(p, ctx->num_sms));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel, p);
}

}  // namespace
}  // namespace kib

using namespace kib;

extern "C" int kib_sample_f32(kib_ctx* ctx, const float* logits, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                              const float* uniform, const float* temperature, const int32_t* top_k, const float* top_p,
                              const float* min_p, int32_t* token_out, float* prob_out, void* stream) {
  KIB_REQUIRE_CTX(ctx);
  KIB_ARG(vocab > 0 && vocab <= (1ull << 23), "sample: vocab must be in 1..2^23");
  KIB_ARG(rows < (1ull << 27), "sample: rows out of range");
  KIB_ARG(row_stride == 0 || (row_stride >= vocab && row_stride < (1ull << 40)), "sample: row stride smaller than a row");
  if (rows == 0) return KIB_OK;
  KIB_ARG(logits && uniform && token_out, "sample: null pointer");
  SampleParams p = {};
  p.logits = logits;
  p.row_stride = static_cast<int64_t>(row_stride ? row_stride : vocab);
  p.rows = static_cast<int>(rows);
  p.vocab = static_cast<int>(vocab);
  p.uniform = uniform;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.token = token_out;
  p.prob = prob_out;
  const cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const cudaError_t e = sample_launch(p, ctx, st);
  if (e != cudaSuccess) return check_cuda(ctx, e, "sample");
  if (!stream) return finish_op(ctx, "sample");
  return check_cuda(ctx, cudaGetLastError(), "sample");
}
