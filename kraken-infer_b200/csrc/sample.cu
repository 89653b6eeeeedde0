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

// ------------------------------------------------------------- by clusters
//
// A cluster of C CTAs takes one row: each CTA keeps its slice of the logits in
// shared memory, so the row is read from HBM once.  One pass turns the logits
// into e_i and, where a cut is wanted, into a histogram of kBins bins over the
// bits of e (32 bins an octave: ordered like e, near-uniform in log e, so a
// vocabulary spreads over hundreds of bins; atomics on one word run one after
// another).  A bin takes two 32-bit shared atomics a logit, its count and the
// sum of the 18 low bits that the bin leaves open: both cuts, and the exact
// mass, follow from them (a slice of 2^14 logits cannot overflow the sum).
// The tokens of the bin with the boundary go to a list, on which two
// histograms of nine bits each narrow the bin to one value of e.  Where a cut
// falls inside a group of equal e, the group is ordered by its logits
// (different logits may round to one e), then by index.  The CTAs add up their
// histograms over distributed shared memory: each adds its non-zero bins to
// share b / (bins / C) of CTA r by remote atomics (integers: in any order the
// same), then everyone gathers the shares and scans them redundantly, one
// cluster barrier a histogram.  Three copies of the small histogram's share
// take turns: a copy is cleared behind the barrier after the one it was
// gathered behind, a barrier before its next use.

constexpr int kSliceMax = 16384;
constexpr int kClusterMax = 16;
constexpr int kClThreads = 512;
constexpr int kBins = 1536;     // 32 an octave: from bin 1281 on e < 2^-40, without weight
constexpr int kBinShift = 18;   // of the bits of e
constexpr int kWeighty = 1281;
constexpr int kFine = 512;      // bins of the histograms on the list
constexpr int kListMax = 2048;
constexpr uint32_t kOneBits = 0x3f800000u;

struct ClusterShared {
  uint32_t cnt[kBins], low[kBins];      // this CTA's histogram
  uint32_t fcnt[kFine], flow[kFine];    // and the small one
  u64 table[kSliceMax / 128];
  u64 scan[kClThreads / 32];
  uint16_t list[kListMax];
  u64 total, before, here;
  float top;
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

__global__ void __launch_bounds__(kClThreads, 2) sample_cluster_kernel(const __grid_constant__ SampleParams p, int slice) {
  extern __shared__ __align__(16) float xs[];  // the slice's logits, then its e; padded with weightless tokens
  float4* x4 = reinterpret_cast<float4*>(xs);
  // shares of the histograms: masses and counts by bin, then three copies of the small one's
  u64* share_mass = reinterpret_cast<u64*>(xs + slice);  // [kBins / C]
  __shared__ ClusterShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const unsigned C = cl.num_blocks(), rank = cl.block_rank();
  const int row = static_cast<int>(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = static_cast<int>(rank) * slice, n = max(0, min(slice, p.vocab - i0));
  const float* x = p.logits + static_cast<int64_t>(row) * p.row_stride + i0;

  const float t = p.temperature ? __ldg(p.temperature + row) : 1.0f;
  const int k = p.top_k ? __ldg(p.top_k + row) : 0;
  const float top_p = p.top_p ? __ldg(p.top_p + row) : 1.0f;
  const float min_p0 = p.min_p ? __ldg(p.min_p + row) : 0.0f;
  const float min_p = min_p0 > 0.0f ? fminf(min_p0, 1.0f) : 0.0f;
  const float u = __ldg(p.uniform + row), inv_t = __fdiv_rn(1.0f, t);
  const int n4 = slice / 4, per = kBins / static_cast<int>(C), fper = kFine / static_cast<int>(C);
  u64* share_fine = share_mass + per;                                     // [3][kFine / C]
  uint32_t* share_cnt = reinterpret_cast<uint32_t*>(share_fine + 3 * fper);  // [kBins / C]

  // the slice, cleaned, and its maximum
  float top = -INFINITY;
  if (i0 + slice <= p.vocab && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll 4
    for (int i = tid; i < n4; i += kClThreads) {
      float4 l = __ldg(reinterpret_cast<const float4*>(x) + i);
      l = make_float4(clean_logit(l.x), clean_logit(l.y), clean_logit(l.z), clean_logit(l.w));
      x4[i] = l;
      top = fmaxf(fmaxf(top, fmaxf(l.x, l.y)), fmaxf(l.z, l.w));
    }
  } else {
#pragma unroll 8
    for (int i = tid; i < slice; i += kClThreads) {
      const float l = i < n ? clean_logit(__ldg(x + i)) : -INFINITY;
      xs[i] = l;
      top = fmaxf(top, l);
    }
  }
  for (int j = tid; j < per; j += kClThreads) share_mass[j] = 0, share_cnt[j] = 0;
  for (int j = tid; j < 3 * fper; j += kClThreads) share_fine[j] = 0;
  top = warp_max(top);
  float* fs = reinterpret_cast<float*>(sh.scan);
  if (lane == 0) fs[warp] = top;
  if (tid == 0) sh.first = 0x7fffffff;
  for (int b = tid; b < kBins; b += kClThreads) sh.cnt[b] = sh.low[b] = 0;
  if (tid < kFine) sh.fcnt[tid] = sh.flow[tid] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kClThreads / 32; ++w) top = fmaxf(top, fs[w]);
    sh.top = top;
  }
  cl.sync();
  top = warp_max(lane < static_cast<int>(C) ? *peer(cl, &sh.top, lane) : -INFINITY);

  if (top == -INFINITY || !(t > 1e-6f)) {
    int best = 0x7fffffff;
    if (top > -INFINITY)
      for (int i = tid; i < n; i += kClThreads)
        if (xs[i] == top) best = min(best, i0 + i);
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0 && best != 0x7fffffff) atomicMin(&sh.first, best);
    cl.sync();
    if (rank == 0 && warp == 0) {
      best = __reduce_min_sync(0xffffffffu, lane < static_cast<int>(C) ? *peer(cl, &sh.first, lane) : 0x7fffffff);
      if (lane == 0) {
        p.token[row] = best == 0x7fffffff ? -1 : best;
        if (p.prob) p.prob[row] = best == 0x7fffffff ? 0.0f : 1.0f;
      }
    }
    cl.sync();
    return;
  }
  const RowScale rs{top, inv_t};
  const bool by_k = k > 0 && k < p.vocab, by_p = !(top_p >= 1.0f);

  auto owner_of = [&](int b) { return static_cast<unsigned>(b) * C / kBins; };  // of a bin's share
  auto e_bits = [&](int i) { return __float_as_uint(xs[i]); };
  auto logit_key = [&](int i) { return order_key(i < n ? clean_logit(__ldg(x + i)) : -INFINITY); };
  auto e_bin = [](uint32_t bits) { return min(static_cast<int>(kOneBits >> kBinShift) - static_cast<int>(bits >> kBinShift), kBins - 1); };
  auto bin_bits = [](int bin) { return ((kOneBits >> kBinShift) - static_cast<uint32_t>(bin)) << kBinShift; };  // its smallest

  // logits to weights: with the histogram on the way, or (no cut to find) the sum of the kept
  const uint32_t min_bits = __float_as_uint(min_p);
  u64 kept_mass = 0;
  for (int i = tid; i < n4; i += kClThreads) {
    const float4 l = x4[i];
    const float e[4] = {logit_weight(l.x, rs), logit_weight(l.y, rs), logit_weight(l.z, rs), logit_weight(l.w, rs)};
    x4[i] = make_float4(e[0], e[1], e[2], e[3]);
    if (by_k || by_p) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = __float_as_uint(e[j]);
        const int bin = e_bin(b);
        atomicAdd(&sh.cnt[bin], 1u);
        atomicAdd(&sh.low[bin], (b & ((1u << kBinShift) - 1)) >> min(low_shift(b), 31));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) kept_mass += __float_as_uint(e[j]) >= min_bits ? fixed_weight(e[j]) : 0;
    }
  }

  // What is kept: bits of e above cut.bits; of those equal to it, all, or
  // (partial) those with a logit key above cut.key, and with it up to index cut.last.
  struct {
    uint32_t bits, key;
    int last;
    bool partial;
  } cut = {0u, 0u, 0x7fffffff, false};
  auto in_cut = [&](int i) {
    const uint32_t b = e_bits(i);
    if (b != cut.bits || !cut.partial) return b >= cut.bits;
    const uint32_t key = logit_key(i);
    return key > cut.key || (key == cut.key && i0 + i <= cut.last);
  };

  // Of the values that a thread holds, in scan order over the threads: sets
  // sh.bin, sh.before, sh.here where the running sum (from `before`) reaches want.
  auto find = [&](const u64* v, auto per_thread, u64 before, u64 acc, u64 want) {
    constexpr int PER = decltype(per_thread)::value;
    acc += before;
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
  auto find_fine = [&](bool masses, uint32_t top_bits, int open, u64* before, u64* here, u64 want) -> int {
    u64* mine_at = share_fine + turn * fper;
    turn = turn == 2 ? 0 : turn + 1;
    __syncthreads();
    {
      const uint32_t count = sh.fcnt[tid];
      u64 v = count;
      if (masses) v = bin_mass(top_bits | static_cast<uint32_t>(kFine - 1 - tid) << open, count, sh.flow[tid]);
      sh.fcnt[tid] = sh.flow[tid] = 0;  // for the next
      if (v) atomicAdd(peer(cl, mine_at + (tid & (fper - 1)), tid * C / kFine), v);
    }
    cl.sync();
    // the copy before last has been gathered by everyone
    for (int j = tid; j < fper; j += kClThreads) share_fine[(turn == 2 ? 0 : turn + 1) * fper + j] = 0;
    const u64 v = *peer(cl, mine_at + (tid & (fper - 1)), tid * C / kFine);
    if (tid == 0) sh.bin = kFine - 1, sh.before = *before, sh.here = 0;
    u64 total;
    const u64 acc = block_scan<kClThreads>(v, sh.scan, &total);
    find(&v, std::integral_constant<int, 1>{}, *before, acc, want);
    *before = sh.before;
    *here = sh.here;
    const int bin = sh.bin;
    __syncthreads();  // sh.bin is written again
    return bin;
  };
  static_assert(kFine == kClThreads, "one bin of the small histogram a thread");
  // The tokens with bits of e in [klo, khi] that `member` lets through, listed;
  // or gone through again and again where the list is too short.
  bool short_list = false;
  auto make_list = [&](uint32_t klo, uint32_t khi, auto member) {
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    for (int q = tid; q < n4; q += kClThreads) {
      const uint4 b = reinterpret_cast<const uint4*>(xs)[q];
      const uint32_t bits[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (bits[j] < klo || bits[j] > khi || !member(4 * q + j)) continue;
        const int at = atomicAdd(&sh.listed, 1);
        if (at < kListMax) sh.list[at] = static_cast<uint16_t>(4 * q + j);
      }
    }
    __syncthreads();
    short_list = sh.listed <= kListMax;
  };
  auto for_list = [&](uint32_t klo, uint32_t khi, auto member, auto what) {
    if (short_list) {
      for (int j = tid; j < sh.listed; j += kClThreads) what(static_cast<int>(sh.list[j]));
    } else {
      for (int i = tid; i < slice; i += kClThreads) {
        const uint32_t b = e_bits(i);
        if (b >= klo && b <= khi && member(i)) what(i);
      }
    }
  };
  // The block's sum, then the cluster's, of a value of each thread.
  auto cluster_sum = [&](u64 v) -> u64 {
    u64 all;
    block_scan<kClThreads>(v, sh.scan, &all);
    if (tid == 0) sh.total = all;
    cl.sync();
    u64 sum = lane < static_cast<int>(C) ? *peer(cl, &sh.total, lane) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };

  // Weights summed in index order: the token (relative to the slice) at which
  // the running sum exceeds aim(total), in the CTA that holds it (-1 in the
  // others); *owner is that CTA's rank.
  // `mine`: this thread's part of the CTA's sum.
  auto locate = [&](u64 mine, auto weight, auto aim_of, unsigned* owner, u64* total) -> int {
    // weight(q, w): the weights of tokens 4 q .. 4 q + 3
    u64 all = 0, w[4];
    block_scan<kClThreads>(mine, sh.scan, &all);
    if (tid == 0) sh.total = all;
    cl.sync();
    const u64 theirs = lane < static_cast<int>(C) ? *peer(cl, &sh.total, lane) : 0;
    u64 inc = theirs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    *total = __shfl_sync(0xffffffffu, inc, 31);
    const u64 aim = aim_of(*total);
    *owner = min(static_cast<unsigned>(__ffs(__ballot_sync(0xffffffffu, inc > aim)) - 1), C - 1);
    const u64 base = __shfl_sync(0xffffffffu, inc - theirs, *owner);
    if (*owner != rank) return -1;
    constexpr int W = kClThreads / 32;
    const int rounds = (n4 + kClThreads - 1) / kClThreads;
    for (int j = 0; j < rounds; ++j) {
      const int q = j * kClThreads + tid;
      u64 v = 0;
      if (q < n4) {
        weight(q, w);
        v = (w[0] + w[1]) + (w[2] + w[3]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) sh.table[j * W + warp] = v;
    }
    if (tid == 0) sh.bin = 0, sh.before = base;
    __syncthreads();
    const u64 v = tid < rounds * W ? sh.table[tid] : 0;
    const u64 acc = base + block_scan<kClThreads>(v, sh.scan, &all);
    if (acc <= aim && aim < acc + v) sh.bin = tid, sh.before = acc;
    __syncthreads();
    const int q = sh.bin / W * kClThreads + sh.bin % W * 32 + lane;
    w[0] = w[1] = w[2] = w[3] = 0;
    if (q < n4) weight(q, w);
    const u64 four = (w[0] + w[1]) + (w[2] + w[3]);
    u64 run = four;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u2 = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u2;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sh.before + run > aim);
    run += sh.before - four;
    int at = 4 * q;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      run += w[j];
      at += run <= aim;
    }
    return __shfl_sync(0xffffffffu, at, max(__ffs(past) - 1, 0));
  };

  // Moves the cut into bin `bin`, of whose tokens (that pass the cut so far,
  // for masses) `before` already lies ahead, to where the sum reaches want.
  auto select = [&](bool masses, int bin, u64 before, u64 want) {
    const uint32_t klo = bin_bits(bin), khi = min(klo + ((1u << kBinShift) - 1), kOneBits);
    auto member = [&](int i) { return !masses || in_cut(i); };
    make_list(klo, khi, member);
    u64 here = 0;
    const int shift = min(low_shift(klo), 31);
    for_list(klo, khi, member, [&](int i) {
      const uint32_t b = e_bits(i);
      const int f = kFine - 1 - static_cast<int>(b >> 9 & 511u);
      atomicAdd(&sh.fcnt[f], 1u);
      if (masses) atomicAdd(&sh.flow[f], (b & 511u) >> shift);
    });
    const uint32_t mid = klo | static_cast<uint32_t>(kFine - 1 - find_fine(masses, klo, 9, &before, &here, want)) << 9;
    for_list(klo, khi, member, [&](int i) {
      const uint32_t b = e_bits(i);
      if (b >> 9 == mid >> 9) atomicAdd(&sh.fcnt[kFine - 1 - static_cast<int>(b & 511u)], 1u);
    });
    const uint32_t bits = mid | static_cast<uint32_t>(kFine - 1 - find_fine(masses, mid, 0, &before, &here, want));
    const u64 w = masses ? max(fixed_weight(__uint_as_float(bits)), 1ull) : 1;
    u64 ties = (want - before + w - 1) / w;
    const bool partial = ties < here / w || (masses && cut.partial && bits == cut.bits);
    cut.bits = bits;
    cut.partial = partial;
    if (!partial) return;
    // the first `ties` of the tokens with this e: by logit, then by index
    auto any = [](int) { return true; };
    if (tid == 0) sh.kmin = 0xffffffffu, sh.kmax = 0;
    make_list(bits, bits, any);
    uint32_t lo = 0xffffffffu, hi = 0;
    for_list(bits, bits, any, [&](int i) {
      const uint32_t key = logit_key(i);
      lo = min(lo, key), hi = max(hi, key);
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) atomicMin(&sh.kmin, lo), atomicMax(&sh.kmax, hi);
    cl.sync();
    lo = __reduce_min_sync(0xffffffffu, lane < static_cast<int>(C) ? *peer(cl, &sh.kmin, lane) : 0xffffffffu);
    hi = __reduce_max_sync(0xffffffffu, lane < static_cast<int>(C) ? *peer(cl, &sh.kmax, lane) : 0u);
    before = 0;
    for (int level = 0; lo < hi && level < 8; ++level) {  // four at most: 2^32 keys, 2^9 a level
      const int open = max(0, 23 - __clz(hi - lo));
      for_list(bits, bits, any, [&](int i) {
        const uint32_t key = logit_key(i);
        if (key >= lo && key <= hi) atomicAdd(&sh.fcnt[(hi - key) >> open], 1u);
      });
      const uint32_t top_key = hi - (static_cast<uint32_t>(find_fine(false, 0u, 0, &before, &here, ties)) << open), size = 1u << open;
      lo = top_key - lo >= size - 1 ? top_key - (size - 1) : lo;
      hi = top_key;
    }
    cut.key = lo;
    ties -= before;
    u64 mine = 0;
    for_list(bits, bits, any, [&](int i) { mine += logit_key(i) == lo; });
    unsigned owner;
    u64 total;
    const int at = locate(
        mine,
        [&](int q, u64(&w4)[4]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w4[j] = e_bits(4 * q + j) == bits && logit_key(4 * q + j) == lo;
        },
        [&](u64) { return ties - 1; }, &owner, &total);
    if (at >= 0 && tid == 0) sh.index = i0 + at;
    cl.sync();
    cut.last = *peer(cl, &sh.index, owner);
  };
  auto kept = [&](int q, u64(&w)[4]) {
    const uint4 b = reinterpret_cast<const uint4*>(xs)[q];
    const uint32_t bits[4] = {b.x, b.y, b.z, b.w};
    const uint32_t low = max(cut.bits, min_bits);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0;
      if (bits[j] >= low && (bits[j] != cut.bits || !cut.partial || in_cut(4 * q + j))) w[j] = fixed_weight(__uint_as_float(bits[j]));
    }
  };
  if (by_k || by_p) {
    // the cluster's bins: three to a thread, in the order of the candidates
    __syncthreads();
    for (int b = tid; b < kBins; b += kClThreads) {
      const uint32_t count = sh.cnt[b];
      if (!count) continue;
      atomicAdd(peer(cl, share_cnt + b - owner_of(b) * per, owner_of(b)), count);
      if (by_p && b < kWeighty) atomicAdd(peer(cl, share_mass + b - owner_of(b) * per, owner_of(b)), bin_mass(bin_bits(b), count, sh.low[b]));
    }
    cl.sync();
    constexpr int PER = kBins / kClThreads;
    u64 mass[PER], sum = 0;
    int k_bin = kBins;  // bins from it on are cut, but for what stays of its own
    u64 k_mass = 0;
    if (by_k) {
      u64 v[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = *peer(cl, share_cnt + b - owner_of(b) * per, owner_of(b));
        sum += v[e];
      }
      u64 total;
      const u64 acc = block_scan<kClThreads>(sum, sh.scan, &total);
      find(v, std::integral_constant<int, PER>{}, 0, acc, static_cast<u64>(k));
      const int bin = sh.bin;
      const u64 before = sh.before;
      __syncthreads();
      if (bin < kWeighty) {  // else every token with weight is kept
        k_bin = bin;
        select(false, bin, before, static_cast<u64>(k));
        if (by_p) {
          // what is kept of its bin (the list may be that of a group of equals by now)
          const uint32_t klo = bin_bits(bin), khi = klo + ((1u << kBinShift) - 1);
          u64 mine = 0;
          for (int q = tid; q < n4; q += kClThreads) {
            const uint4 b = reinterpret_cast<const uint4*>(xs)[q];
            const uint32_t bits[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (bits[j] >= cut.bits && bits[j] >= klo && bits[j] <= khi && in_cut(4 * q + j)) mine += fixed_weight(__uint_as_float(bits[j]));
          }
          k_mass = cluster_sum(mine);
        }
      }
    }
    if (by_p) {
      sum = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        mass[e] = b < k_bin ? *peer(cl, share_mass + b - owner_of(b) * per, owner_of(b)) : (b == k_bin ? k_mass : 0);
        sum += mass[e];
      }
      u64 total;
      const u64 acc = block_scan<kClThreads>(sum, sh.scan, &total);
      const double limit = static_cast<double>(total) * static_cast<double>(top_p);
      const u64 want = limit > 1.0 ? static_cast<u64>(limit) : 1ull;
      find(mass, std::integral_constant<int, PER>{}, 0, acc, want);
      const int bin = sh.bin;
      const u64 before = sh.before;
      __syncthreads();
      select(true, bin, before, want);
    }
    // this CTA's kept mass: whole bins from its histogram, the cut's own token by token
    const uint32_t low = max(cut.bits, min_bits);
    const int edge = e_bin(low);
    for (int b = tid; b < min(edge, kWeighty); b += kClThreads) kept_mass += bin_mass(bin_bits(b), sh.cnt[b], sh.low[b]);
    if (edge < kWeighty) {
      const uint32_t khi = min(bin_bits(edge) + ((1u << kBinShift) - 1), kOneBits);
      for (int q = tid; q < n4; q += kClThreads) {
        const uint4 b = reinterpret_cast<const uint4*>(xs)[q];
        const uint32_t bits[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bits[j] >= low && bits[j] <= khi && (bits[j] != cut.bits || !cut.partial || in_cut(4 * q + j)))
            kept_mass += fixed_weight(__uint_as_float(bits[j]));
      }
    }
  }

  unsigned owner;
  u64 total;
  const int token = locate(kept_mass, kept,
                           [&](u64 all) -> u64 {
                             const double f = static_cast<double>(all) * static_cast<double>(u);
                             return f > 0.0 ? min(static_cast<u64>(f), all - 1) : 0;
                           },
                           &owner, &total);
  if (token >= 0 && tid == 0) {
    p.token[row] = i0 + token;
    if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(fixed_weight(xs[token])) / static_cast<double>(total));
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

// ------------------------------------------------------------------ by rows
//
// One CTA takes a row and reads it three times, mostly from L2: its maximum;
// the histogram, as above; and, in warps' segments of the index order, what is
// kept.  No cluster barriers and one set of scans a row, so it does the same
// work in a third of the time where rows fill the GPU, and it takes rows of
// any length; a single row is faster on a cluster.  The histogram's sums of
// low bits are folded into 64-bit masses every 2^14 logits, before they can
// overflow.

// (two CTAs of 512 threads an SM took 376 us for 256 rows of 248320, one of 1024 330 us)
constexpr int kRowThreads = 1024;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowList = 4096;

struct RowShared {
  uint32_t cnt[kBins], low[kBins];
  u64 mass[kBins];
  uint32_t count[kBins];
  uint32_t fcnt[kFine], flow[kFine];
  u64 scan[kRowWarps];
  uint32_t list[kRowList], list_bits[kRowList];
  u64 segment[kRowWarps];
  u64 before, here;
  float top[kRowWarps];
  int first, bin, listed, index;
  uint32_t kmin, kmax;
};

__global__ void __launch_bounds__(kRowThreads, 1) sample_row_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t row_raw[];
  RowShared& sh = *reinterpret_cast<RowShared*>(row_raw);
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.vocab, Q = (V + 3) / 4;
  const float* x = p.logits + static_cast<int64_t>(row) * p.row_stride;
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const float t = p.temperature ? __ldg(p.temperature + row) : 1.0f;
  const int k = p.top_k ? __ldg(p.top_k + row) : 0;
  const float top_p = p.top_p ? __ldg(p.top_p + row) : 1.0f;
  const float min_p0 = p.min_p ? __ldg(p.min_p + row) : 0.0f;
  const float min_p = min_p0 > 0.0f ? fminf(min_p0, 1.0f) : 0.0f;
  const float u = __ldg(p.uniform + row), inv_t = __fdiv_rn(1.0f, t);
  // logits below it cannot be among the first k: read as -infinity
  float least = -INFINITY;
  auto clean = [&](float l) {
    l = clean_logit(l);
    return l < least ? -INFINITY : l;
  };
  auto load = [&](int q) -> float4 {
    float4 l;
    if (wide && 4 * q + 3 < V) {
      l = __ldg(reinterpret_cast<const float4*>(x) + q);
    } else {
      l.x = 4 * q < V ? __ldg(x + 4 * q) : -INFINITY;
      l.y = 4 * q + 1 < V ? __ldg(x + 4 * q + 1) : -INFINITY;
      l.z = 4 * q + 2 < V ? __ldg(x + 4 * q + 2) : -INFINITY;
      l.w = 4 * q + 3 < V ? __ldg(x + 4 * q + 3) : -INFINITY;
    }
    return make_float4(clean(l.x), clean(l.y), clean(l.z), clean(l.w));
  };

  // four quads, `step` apart, all asked for before the first is used
  auto load_four = [&](int q, int step, int end, float4 (&l)[4]) {
    if (wide && q + 3 * step < min(end, V / 4)) {
#pragma unroll
      for (int w = 0; w < 4; ++w) l[w] = __ldg(reinterpret_cast<const float4*>(x) + q + w * step);
#pragma unroll
      for (int w = 0; w < 4; ++w) l[w] = make_float4(clean(l[w].x), clean(l[w].y), clean(l[w].z), clean(l[w].w));
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        l[w] = q + w * step < end ? load(q + w * step) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
  };

  float top = -INFINITY;
  for (int q = tid; q < Q; q += 4 * kRowThreads) {
    float4 l[4];
    load_four(q, kRowThreads, Q, l);
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(fmaxf(top, fmaxf(l[w].x, l[w].y)), fmaxf(l[w].z, l[w].w));
  }
  const float own_top = top;
  top = warp_max(top);
  if (lane == 0) sh.top[warp] = top;
  if (tid == 0) sh.first = 0x7fffffff, sh.index = 0, sh.listed = 0;
  for (int b = tid; b < kBins; b += kRowThreads) sh.cnt[b] = sh.low[b] = sh.count[b] = 0, sh.mass[b] = 0;
  if (tid < kFine) sh.fcnt[tid] = sh.flow[tid] = 0;
  __syncthreads();
  top = warp_max(lane < kRowWarps ? sh.top[lane] : -INFINITY);

  if (top == -INFINITY || !(t > 1e-6f)) {
    int best = 0x7fffffff;
    if (top > -INFINITY)
      for (int q = tid; q < Q; q += kRowThreads) {
        const float4 l = load(q);
        const int at = l.x == top ? 0 : (l.y == top ? 1 : (l.z == top ? 2 : (l.w == top ? 3 : 4)));
        if (at < 4) best = min(best, 4 * q + at);
      }
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0 && best != 0x7fffffff) atomicMin(&sh.first, best);
    __syncthreads();
    if (tid == 0) {
      p.token[row] = sh.first == 0x7fffffff ? -1 : sh.first;
      if (p.prob) p.prob[row] = sh.first == 0x7fffffff ? 0.0f : 1.0f;
    }
    return;
  }
  const RowScale rs{top, inv_t};
  const bool by_k = k > 0 && k < V, by_p = !(top_p >= 1.0f);
  const uint32_t min_bits = __float_as_uint(min_p);
  // k of the threads' maxima are k tokens, so the k-th token is no less than
  // the k-th maximum (16 bits of it, found bit by bit): of a long row a few
  // more than k tokens are left, and all else works on their list
  if (by_k && k <= kRowThreads) {
    const uint32_t key = order_key(own_top) >> 16;
    uint32_t at = 0;
    for (int bit = 15; bit >= 0; --bit)
      if (__syncthreads_count(key >= (at | 1u << bit)) >= k) at |= 1u << bit;
    at <<= 16;
    least = __uint_as_float(at & 0x80000000u ? at ^ 0x80000000u : ~at);  // below -infinity's: a NaN, which hides nothing
  }
  const bool hidden = least > -INFINITY;
  bool all_listed = false;
  auto bits_at = [&](int i) { return __float_as_uint(logit_weight(clean_logit(__ldg(x + i)), rs)); };
  auto logit_key = [&](int i) { return order_key(clean_logit(__ldg(x + i))); };
  auto e_bin = [](uint32_t bits) { return min(static_cast<int>(kOneBits >> kBinShift) - static_cast<int>(bits >> kBinShift), kBins - 1); };
  auto bin_bits = [](int bin) { return ((kOneBits >> kBinShift) - static_cast<uint32_t>(bin)) << kBinShift; };
  // what of (l - top) / T a token with these bits of e has at least (at most): spares the exponential of the others
  auto z_of = [&](float l) { return __fmul_rn(l == rs.top ? 0.0f : __fsub_rn(l, rs.top), rs.inv_t); };
  auto z_floor = [](uint32_t bits) { return bits ? logf(__uint_as_float(bits)) - 1e-4f : -INFINITY; };

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
  auto find = [&](const u64* v, auto per_thread, u64 acc, u64 want) {
    constexpr int PER = decltype(per_thread)::value;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (acc < want && want <= acc + v[e]) sh.bin = tid * PER + e, sh.before = acc, sh.here = v[e];
      acc += v[e];
    }
    __syncthreads();
  };
  auto find_fine = [&](bool masses, uint32_t top_bits, int open, u64* before, u64* here, u64 want) -> int {
    __syncthreads();
    u64 v = 0;
    if (tid < kFine) {
      const uint32_t count = sh.fcnt[tid];
      v = masses ? bin_mass(top_bits | static_cast<uint32_t>(kFine - 1 - tid) << open, count, sh.flow[tid]) : count;
      sh.fcnt[tid] = sh.flow[tid] = 0;
    }
    if (tid == 0) sh.bin = kFine - 1, sh.before = *before, sh.here = 0;
    u64 total;
    const u64 acc = *before + block_scan<kRowThreads>(v, sh.scan, &total);
    find(&v, std::integral_constant<int, 1>{}, acc, want);
    *before = sh.before;
    *here = sh.here;
    const int bin = sh.bin;
    __syncthreads();
    return bin;
  };
  // The tokens with bits of e in [klo, khi]: listed, or gone through where there are too many.
  auto for_range = [&](uint32_t klo, uint32_t khi, auto what) {
    const float zl = z_floor(klo), zh = khi >= kOneBits ? INFINITY : logf(__uint_as_float(max(khi, 1u))) + 1e-4f;
    for (int q0 = tid; q0 < Q; q0 += 4 * kRowThreads) {
      float4 l4[4];
      load_four(q0, kRowThreads, Q, l4);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float l[4] = {l4[w].x, l4[w].y, l4[w].z, l4[w].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float z = z_of(l[j]);
          if (!(z >= zl && z <= zh)) continue;
          const int i = 4 * (q0 + w * kRowThreads) + j;
          const uint32_t b = __float_as_uint(logit_weight(l[j], rs));
          if (b >= klo && b <= khi && i < V) what(i, b);
        }
      }
    }
  };
  bool short_list = false;
  auto make_list = [&](uint32_t klo, uint32_t khi) {
    if (all_listed) return;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    for_range(klo, khi, [&](int i, uint32_t b) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kRowList) sh.list[at] = static_cast<uint32_t>(i), sh.list_bits[at] = b;
    });
    __syncthreads();
    short_list = sh.listed <= kRowList;
  };
  auto for_list = [&](uint32_t klo, uint32_t khi, auto what) {
    if (short_list) {
      for (int j = tid; j < sh.listed; j += kRowThreads)
        if (sh.list_bits[j] >= klo && sh.list_bits[j] <= khi) what(static_cast<int>(sh.list[j]), sh.list_bits[j]);
    } else {
      for_range(klo, khi, what);
    }
  };
  // Index at which the running sum, in index order, of weight(i, bits of e)
  // over the tokens with bits of at least `floor` exceeds aim_of(total): the
  // warps' segments first, then the block goes through the one that holds it.
  auto locate = [&](uint32_t floor, auto weight, auto aim_of, u64* total) -> int {
    const float zl = z_floor(floor);
    const int s0 = static_cast<int>(static_cast<int64_t>(Q) * warp / kRowWarps), s1 = static_cast<int>(static_cast<int64_t>(Q) * (warp + 1) / kRowWarps);
    auto four = [&](int q, const float4& l4, u64 (&w)[4]) {
      const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
        if (!(z_of(l[j]) >= zl) || 4 * q + j >= V) continue;
        const uint32_t b = __float_as_uint(logit_weight(l[j], rs));
        if (b >= floor) w[j] = weight(4 * q + j, b);
      }
    };
    u64 sum = 0, w[4];
    __syncthreads();
    if (all_listed) {
      if (tid < kRowWarps) sh.segment[tid] = 0;
      __syncthreads();
      for (int j = tid; j < sh.listed; j += kRowThreads) {
        const int i = static_cast<int>(sh.list[j]);
        const u64 v = sh.list_bits[j] >= floor ? weight(i, sh.list_bits[j]) : 0;
        if (v) atomicAdd(&sh.segment[(32 * (i / 4 + 1) - 1) / Q], v);  // the segment that holds quad i / 4
      }
    }
    for (int q = all_listed ? s1 : s0 + lane; q < s1; q += 128) {
      float4 l4[4];
      load_four(q, 32, s1, l4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        four(q + 32 * r, l4[r], w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0 && !all_listed) sh.segment[warp] = sum;
    __syncthreads();
    u64 base = 0, all = 0;
    int seg = kRowWarps - 1;
    for (int s = 0; s < kRowWarps; ++s) all += sh.segment[s];
    *total = all;
    const u64 aim = aim_of(all);
    for (int s = 0; s < kRowWarps; ++s) {
      if (aim < base + sh.segment[s]) {
        seg = s;
        break;
      }
      base += sh.segment[s];
    }
    const int q0 = static_cast<int>(static_cast<int64_t>(Q) * seg / kRowWarps), q1 = static_cast<int>(static_cast<int64_t>(Q) * (seg + 1) / kRowWarps);
    for (int qb = q0; qb < q1; qb += kRowThreads) {
      const int q = qb + tid;
      w[0] = w[1] = w[2] = w[3] = 0;
      if (q < q1) four(q, load(q), w);
      const u64 own = (w[0] + w[1]) + (w[2] + w[3]);
      u64 block;
      u64 run = base + block_scan<kRowThreads>(own, sh.scan, &block);
      if (run <= aim && aim < run + own) {
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
    __syncthreads();
    lo = sh.kmin, hi = sh.kmax;
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
    u64 total;
    cut.last = locate(bits, [&](int i, uint32_t b) -> u64 { return b == bits && logit_key(i) == lo; }, [&](u64) { return ties - 1; }, &total);
    __syncthreads();  // sh.index is written again
  };

  if (by_k || by_p) {
    for (int q0 = 0; q0 < Q; q0 += 4 * kRowThreads) {  // 2^14 logits between two folds
      float4 l4[4];
      load_four(q0 + tid, kRowThreads, Q, l4);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (q0 + tid + w * kRowThreads >= Q) continue;
        const float l[4] = {l4[w].x, l4[w].y, l4[w].z, l4[w].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (hidden && l[j] == -INFINITY) continue;
          const uint32_t b = __float_as_uint(logit_weight(l[j], rs));
          const int bin = e_bin(b);
          if (hidden) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < kRowList) sh.list[at] = static_cast<uint32_t>(4 * (q0 + tid + w * kRowThreads) + j), sh.list_bits[at] = b;
          }
          atomicAdd(&sh.cnt[bin], 1u);
          atomicAdd(&sh.low[bin], (b & ((1u << kBinShift) - 1)) >> min(low_shift(b), 31));
        }
      }
      __syncthreads();
      for (int b = tid; b < kBins; b += kRowThreads) {
        const uint32_t count = sh.cnt[b];
        if (!count) continue;
        sh.count[b] += count;
        if (b < kWeighty) sh.mass[b] += bin_mass(bin_bits(b), count, sh.low[b]);
        sh.cnt[b] = sh.low[b] = 0;
      }
      __syncthreads();
    }
    if (hidden && sh.listed <= kRowList) all_listed = short_list = true;
    constexpr int PER = (kBins + kRowThreads - 1) / kRowThreads;
    u64 v[PER], sum = 0, total;
    int k_bin = kBins;
    u64 k_mass = 0;
    if (by_k) {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = b < kBins ? sh.count[b] : 0;
        sum += v[e];
      }
      const u64 acc = block_scan<kRowThreads>(sum, sh.scan, &total);
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
          block_scan<kRowThreads>(mine, sh.scan, &k_mass);
        }
      }
    }
    if (by_p) {
      sum = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = b < min(k_bin, kBins) ? sh.mass[b] : (b == k_bin ? k_mass : 0);
        sum += v[e];
      }
      const u64 acc = block_scan<kRowThreads>(sum, sh.scan, &total);
      const double limit = static_cast<double>(total) * static_cast<double>(top_p);
      const u64 want = limit > 1.0 ? static_cast<u64>(limit) : 1ull;
      find(v, std::integral_constant<int, PER>{}, acc, want);
      const int bin = sh.bin;
      const u64 before = sh.before;
      __syncthreads();
      select(true, bin, before, want);
    }
  }
  u64 total;
  const uint32_t floor = max(cut.bits, min_bits);
  const int token = locate(floor,
                           [&](int i, uint32_t b) -> u64 {
                             return b != cut.bits || !cut.partial || in_cut(i, b) ? fixed_weight(__uint_as_float(b)) : 0;
                           },
                           [&](u64 all) -> u64 {
                             const double f = static_cast<double>(all) * static_cast<double>(u);
                             return f > 0.0 ? min(static_cast<u64>(f), all - 1) : 0;
                           },
                           &total);
  if (tid == 0) {
    p.token[row] = token;
    if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(fixed_weight(__uint_as_float(bits_at(token)))) / static_cast<double>(total));
  }
}

// The fewest CTAs that hold a row in shared memory.
int cluster_of(int vocab) {
  int c = 1;
  while (c * kSliceMax < vocab) c *= 2;
  return c;
}
// A row whose logits one CTA holds is always fastest there.  Longer ones take
// clusters while those of about five rounds cover the GPU: measured at 248320
// tokens 64 rows 157 us by clusters and 178 by rows, 96 rows 232 and 190, 256
// rows 587 and 330; at 100000 tokens 64 rows 61 and 100, 256 rows 216 and 150.
bool by_rows(const SampleParams& p, int num_sms) {
  const int c = cluster_of(p.vocab);
  return c > kClusterMax || (c > 1 && static_cast<int64_t>(p.rows) * c > 8ll * num_sms);
}

cudaError_t sample_cluster_launch(const SampleParams& p, int num_sms, cudaStream_t st) {
  static bool ready = false;
  cudaError_t e;
  if (!ready) {
    e = cudaFuncSetAttribute(sample_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceMax * 4 + kBins * 12 + kFine * 24);
    pin_carveout(sample_cluster_kernel);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    ready = true;
  }
  // for few rows more CTAs than hold one, down to slices of 2048
  int c = cluster_of(p.vocab);
  while (c < kClusterMax && static_cast<int64_t>(p.rows) * c * 2 <= num_sms && p.vocab / (2 * c) >= 2048) c *= 2;
  const int slice = ((p.vocab + c - 1) / c + 127) / 128 * 128;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * static_cast<unsigned>(c));
  cfg.blockDim = dim3(kClThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(slice) * sizeof(float) + (kBins * 12 + kFine * 24) / c;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(c);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_cluster_kernel, p, slice);
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
  cudaError_t e;
  if (!by_rows(p, ctx->num_sms)) {
    e = sample_cluster_launch(p, ctx->num_sms, st);
  } else {
    static bool ready = false;
    e = ready ? cudaSuccess
              : cudaFuncSetAttribute(sample_row_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(RowShared)));
    ready = e == cudaSuccess;
    if (ready) sample_row_kernel<<<static_cast<unsigned>(rows), kRowThreads, sizeof(RowShared), st>>>(p);
  }
  if (e != cudaSuccess) return check_cuda(ctx, e, "sample");
  if (!stream) return finish_op(ctx, "sample");
  return check_cuda(ctx, cudaGetLastError(), "sample");
}
