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

constexpr int kSampleThreads = 1024;
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
  // +infinity on top: only such logits have weight
  if (l == -INFINITY) return 0.0f;
  const float z = l == r.top ? 0.0f : __fmul_rn(__fsub_rn(l, r.top), r.inv_t);
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

template <typename T, typename Op>
KIB_DEV T block_reduce(T v, Op op, T* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) s[warp] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < kSampleThreads / 32; ++w) v = op(v, s[w]);
  return v;
}

// The end of a prefix in candidate order: keys above `key`, and the first
// `ties` tokens (in index order) with exactly that key.
struct Cut {
  uint32_t key;
  int ties;
};

__global__ void __launch_bounds__(kSampleThreads) sample_row_kernel(const __grid_constant__ SampleParams p) {
  __shared__ float s_f[32];
  __shared__ u64 s_u[32];
  __shared__ int s_i[32];
  __shared__ unsigned s_count[256];
  __shared__ u64 s_mass[256];
  __shared__ uint32_t s_prefix;
  __shared__ u64 s_before;
  const int row = blockIdx.x, tid = threadIdx.x, V = p.vocab;
  const float* x = p.logits + static_cast<int64_t>(row) * p.row_stride;
  auto maxf = [](float a, float b) { return fmaxf(a, b); };
  auto mini = [](int a, int b) { return a < b ? a : b; };
  auto addu = [](u64 a, u64 b) { return a + b; };

  float top = -INFINITY;
  for (int i = tid; i < V; i += kSampleThreads) top = fmaxf(top, clean_logit(x[i]));
  top = block_reduce(top, maxf, s_f);
  if (top == -INFINITY) {  // nothing to choose from
    if (tid == 0) {
      p.token[row] = -1;
      if (p.prob) p.prob[row] = 0.0f;
    }
    return;
  }
  const float t = p.temperature ? p.temperature[row] : 1.0f;
  if (!(t > 1e-6f)) {
    int best = V;
    for (int i = tid; i < V; i += kSampleThreads)
      if (clean_logit(x[i]) == top) best = min(best, i);
    best = block_reduce(best, mini, s_i);
    if (tid == 0) {
      p.token[row] = best;
      if (p.prob) p.prob[row] = 1.0f;
    }
    return;
  }
  const RowScale rs{top, __fdiv_rn(1.0f, t)};
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  const float min_p = p.min_p && p.min_p[row] > 0.0f ? fminf(p.min_p[row], 1.0f) : 0.0f;

  // radix selection of a cut, eight bits of the key at a time: by_count: the
  // cut that keeps `want` tokens; otherwise the shortest prefix whose mass
  // (within `in`) reaches `want`.
  auto select = [&](bool by_count, u64 want, const Cut& in) -> Cut {
    uint32_t prefix = 0;
    u64 before = 0;
    u64 weight = 1;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int b = tid; b < 256; b += kSampleThreads) s_count[b] = 0, s_mass[b] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
        const float l = clean_logit(x[i]);
        const uint32_t key = order_key(l);
        if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        if (by_count) atomicAdd(&s_count[(key >> shift) & 255], 1u);
        else if (key >= in.key) atomicAdd(&s_mass[(key >> shift) & 255], fixed_weight(logit_weight(l, rs)));
      }
      __syncthreads();
      if (tid == 0) {
        u64 acc = before;
        int b = 255;
        for (; b > 0; --b) {
          u64 h = by_count ? s_count[b] : s_mass[b];
          // ties of the enclosing cut beyond its count carry no mass
          if (acc + h >= want) break;
          acc += h;
        }
        s_prefix = prefix | (static_cast<uint32_t>(b) << shift);
        s_before = acc;
      }
      __syncthreads();
      prefix = s_prefix;
      before = s_before;
    }
    if (!by_count) {
      // every token of one key has one weight
      const uint32_t b = prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix;
      weight = fixed_weight(logit_weight(__uint_as_float(b), rs));
    }
    Cut c;
    c.key = prefix;
    const u64 left = want > before ? want - before : 1;
    const u64 n = weight ? (left + weight - 1) / weight : 1;
    c.ties = n > 0x7fffffffull ? 0x7fffffff : static_cast<int>(n);
    if (!by_count && c.key == in.key) c.ties = min(c.ties, in.ties);
    return c;
  };

  Cut cut{0u, 0x7fffffff};  // everything
  if (k > 0 && k < V) cut = select(true, static_cast<u64>(k), cut);
  if (top_p < 1.0f) {
    // mass of the prefix so far
    u64 mass = 0, tied = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float l = clean_logit(x[i]);
      const uint32_t key = order_key(l);
      if (key > cut.key) mass += fixed_weight(logit_weight(l, rs));
      else if (key == cut.key) ++tied;
    }
    mass = block_reduce(mass, addu, s_u);
    tied = block_reduce(tied, addu, s_u);
    if (tied > static_cast<u64>(cut.ties)) tied = static_cast<u64>(cut.ties);
    const uint32_t b = cut.key & 0x80000000u ? cut.key & 0x7fffffffu : ~cut.key;
    if (tied) mass += tied * fixed_weight(logit_weight(__uint_as_float(b), rs));
    double limit = static_cast<double>(mass) * static_cast<double>(top_p);
    u64 want = limit > 1.0 ? static_cast<u64>(limit) : 1;
    if (!(limit == limit)) want = 1;
    cut = select(false, want, cut);
  }

  // kept weights in index order: thread chunks, then a scan of the chunks
  const int chunk = (V + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(tid * chunk, V), i1 = min(i0 + chunk, V);
  int tied = 0;
  for (int i = i0; i < i1; ++i) tied += order_key(clean_logit(x[i])) == cut.key;
  auto scan = [&](u64 v, u64* total) -> u64 {  // exclusive
    const int lane = tid & 31, warp = tid >> 5;
    u64 inc = v;
    for (int o = 1; o < 32; o <<= 1) {
      const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    __syncthreads();
    if (lane == 31) s_u[warp] = inc;
    __syncthreads();
    u64 base = 0, all = 0;
    for (int w = 0; w < kSampleThreads / 32; ++w) {
      if (w < warp) base += s_u[w];
      all += s_u[w];
    }
    *total = all;
    return base + inc - v;
  };
  u64 total = 0;
  const int tie0 = static_cast<int>(min(scan(static_cast<u64>(tied), &total), static_cast<u64>(0x7fffffff)));
  auto kept = [&](int i, int& tie) -> u64 {
    const float l = clean_logit(x[i]);
    const uint32_t key = order_key(l);
    if (key < cut.key || (key == cut.key && tie++ >= cut.ties)) return 0;
    const float e = logit_weight(l, rs);
    return e >= min_p || l == top ? fixed_weight(e) : 0;
  };
  u64 mine = 0;
  int tie = tie0;
  for (int i = i0; i < i1; ++i) mine += kept(i, tie);
  u64 run = scan(mine, &total);
  double aimf = static_cast<double>(total) * static_cast<double>(p.uniform[row]);
  u64 aim = aimf > 0.0 ? static_cast<u64>(aimf) : 0;
  if (aim >= total) aim = total - 1;
  if (run <= aim && aim < run + mine) {
    tie = tie0;
    for (int i = i0; i < i1; ++i) {
      const u64 w = kept(i, tie);
      run += w;
      if (run > aim) {
        p.token[row] = i;
        if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
        break;
      }
    }
  }
}

// ------------------------------------------------------------- by clusters
//
// A cluster of C CTAs takes one row: each CTA keeps its slice of the logits in
// shared memory, so the row is read from HBM once, and every later pass runs
// out of shared memory.  Cuts are found by histograms of kBins bins: the first
// over z = (l - M) / T, which spreads the logits evenly (the leading bits of
// a float would put most of a vocabulary in a few bins, and atomics on one
// word run one after another), the next over the order keys inside the bin
// that holds the boundary, until a bin is one key.  Counts take one 32-bit
// shared atomic a logit, masses the non-zero ones of three (14 + 14 + 12
// bits: a slice of 2^14 logits cannot overflow a word).  The CTAs add up their
// histograms over distributed shared memory: CTA r sums share r of the bins,
// then everyone gathers the sums and scans them redundantly.

constexpr int kSliceMax = 16384;
constexpr int kClusterMax = 16;
constexpr int kClThreads = 512;
constexpr int kBins = 1024;
constexpr float kBinsPerZ = kBins / 28.0f;  // below z = -28 every weight is 0 (2^-40 = e^-27.7)

struct ClusterShared {
  uint32_t hist[3][kBins];
  u64 share[kBins];  // this CTA's summed bins (kBins / C of them)
  u64 sums[kBins];   // all of them, gathered
  u64 scan[kClThreads / 32];
  u64 total;
  float top;
  int first;
  uint32_t kmin, kmax;
  int index;
  u64 before;
  int bin;
};

template <typename T>
KIB_DEV T* peer(cg::cluster_group& cl, T* p, unsigned rank) {
  return cl.map_shared_rank(p, rank);
}

// Exclusive scan over the block; *total gets the sum.
KIB_DEV u64 block_scan(u64 v, u64* s, u64* total) {
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
  u64 base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kClThreads / 32; ++w) {
    if (w < warp) base += s[w];
    all += s[w];
  }
  *total = all;
  return base + inc - v;
}

__global__ void __launch_bounds__(kClThreads, 2) sample_cluster_kernel(const __grid_constant__ SampleParams p, int slice) {
  extern __shared__ __align__(16) float xs[];
  __shared__ ClusterShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const unsigned C = cl.num_blocks(), rank = cl.block_rank();
  const int row = static_cast<int>(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = static_cast<int>(rank) * slice, n = max(0, min(slice, p.vocab - i0));
  const float* x = p.logits + static_cast<int64_t>(row) * p.row_stride + i0;

  // the slice, cleaned, and its maximum
  float top = -INFINITY;
#pragma unroll 8
  for (int i = tid; i < n; i += kClThreads) {
    const float l = clean_logit(__ldg(x + i));
    xs[i] = l;
    top = fmaxf(top, l);
  }
  top = warp_max(top);
  float* fs = reinterpret_cast<float*>(sh.scan);
  if (lane == 0) fs[warp] = top;
  if (tid == 0) sh.first = 0x7fffffff;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kClThreads / 32; ++w) top = fmaxf(top, fs[w]);
    sh.top = top;
  }
  cl.sync();
  top = warp_max(lane < static_cast<int>(C) ? *peer(cl, &sh.top, lane) : -INFINITY);

  const float t = p.temperature ? p.temperature[row] : 1.0f;
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
  const RowScale rs{top, __fdiv_rn(1.0f, t)};
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  const float min_p = p.min_p && p.min_p[row] > 0.0f ? fminf(p.min_p[row], 1.0f) : 0.0f;
  auto key_logit = [](uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); };
  auto z_bin = [&](float l) {
    if (l == rs.top) return 0;
    const float z = __fmul_rn(__fsub_rn(rs.top, l), rs.inv_t) * kBinsPerZ;
    return z < kBins - 1 ? static_cast<int>(z) : kBins - 1;
  };

  Cut cut{0u, 0x7fffffff};
  bool partial = false;  // the cut keeps only some of the tokens with its key
  // One selection: by count (the first `want` tokens) or by mass (the shortest
  // prefix of what `cut` keeps that reaches the fraction top_p of its mass).
  auto select = [&](bool by_count, u64 want) {
    const Cut in = cut;
    const u64 in_tied = by_count || in.key == 0 ? 0 : static_cast<u64>(in.ties) * fixed_weight(logit_weight(key_logit(in.key), rs));
    u64 before = 0;
    uint32_t klo = 0, khi = 0xffffffffu;  // the keys that are left
    int level = 0, shift = 0;
    for (;;) {
      for (int b = tid; b < kBins; b += kClThreads) sh.hist[0][b] = sh.hist[1][b] = sh.hist[2][b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kClThreads) {
        const float l = xs[i];
        const uint32_t key = order_key(l);
        if (key < klo || key > khi) continue;
        if (!by_count && key <= in.key) continue;
        const int b = level == 0 ? z_bin(l) : static_cast<int>((khi - key) >> shift);
        if (by_count) {
          atomicAdd(&sh.hist[0][b], 1u);
        } else {
          const u64 w = fixed_weight(logit_weight(l, rs));
          const uint32_t w0 = static_cast<uint32_t>(w) & 0x3fffu, w1 = static_cast<uint32_t>(w >> 14) & 0x3fffu,
                         w2 = static_cast<uint32_t>(w >> 28);
          if (w0) atomicAdd(&sh.hist[0][b], w0);
          if (w1) atomicAdd(&sh.hist[1][b], w1);
          if (w2) atomicAdd(&sh.hist[2][b], w2);
        }
      }
      cl.sync();
      const int per = kBins / static_cast<int>(C), b0 = static_cast<int>(rank) * per;
      for (int j = tid; j < per; j += kClThreads) {
        u64 v = 0;
        for (unsigned r = 0; r < C; ++r) {
          const uint32_t* h = peer(cl, &sh.hist[0][0], r);
          v += h[b0 + j];
          if (!by_count) v += (static_cast<u64>(h[kBins + b0 + j]) << 14) + (static_cast<u64>(h[2 * kBins + b0 + j]) << 28);
        }
        sh.share[j] = v;
      }
      cl.sync();
      for (int b = tid; b < kBins; b += kClThreads) sh.sums[b] = *peer(cl, &sh.share[b % per], static_cast<unsigned>(b / per));
      __syncthreads();
      constexpr int PER = kBins / kClThreads;
      u64 v[PER], mine = 0, total = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = sh.sums[tid * PER + e], mine += v[e];
      u64 acc = before + block_scan(mine, sh.scan, &total);
      if (level == 0 && !by_count) {
        const double limit = static_cast<double>(total + in_tied) * static_cast<double>(top_p);
        want = limit > 1.0 ? static_cast<u64>(limit) : 1;
        if (total < want) {  // the boundary lies among the ties of the enclosing cut
          const u64 w = fixed_weight(logit_weight(key_logit(in.key), rs));
          const int ties = static_cast<int>(min((want - total + w - 1) / w, static_cast<u64>(in.ties)));
          partial = partial || ties < in.ties;
          cut.ties = ties;
          return;
        }
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (acc < want && want <= acc + v[e]) sh.bin = tid * PER + e, sh.before = acc;
        acc += v[e];
      }
      __syncthreads();
      const int bin = sh.bin;
      before = sh.before;
      const u64 here = sh.sums[bin];
      if (level == 0) {
        // the range of keys in the bin
        uint32_t lo = 0xffffffffu, hi = 0;
        for (int i = tid; i < n; i += kClThreads) {
          const float l = xs[i];
          const uint32_t key = order_key(l);
          if ((by_count || key > in.key) && z_bin(l) == bin) lo = min(lo, key), hi = max(hi, key);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (tid == 0) sh.kmin = 0xffffffffu, sh.kmax = 0;
        __syncthreads();
        if (lane == 0) atomicMin(&sh.kmin, lo), atomicMax(&sh.kmax, hi);
        cl.sync();
        klo = __reduce_min_sync(0xffffffffu, lane < static_cast<int>(C) ? *peer(cl, &sh.kmin, lane) : 0xffffffffu);
        khi = __reduce_max_sync(0xffffffffu, lane < static_cast<int>(C) ? *peer(cl, &sh.kmax, lane) : 0u);
      } else {
        // bin = (khi - key) >> shift
        const uint32_t h = khi - (static_cast<uint32_t>(bin) << shift);
        const uint32_t size = 1u << shift;
        klo = h - klo >= size - 1 ? h - (size - 1) : klo;
        khi = h;
      }
      if (klo >= khi || level == 8) {  // at most five levels: 2^32 keys, 2^10 a level
        const u64 w = by_count ? 1 : max(fixed_weight(logit_weight(key_logit(klo), rs)), 1ull);
        const u64 ties = (want - before + w - 1) / w, group = here / w;
        cut.key = klo;
        cut.ties = static_cast<int>(ties);
        partial = ties < group;
        return;
      }
      ++level;
      const uint32_t range = khi - klo;
      shift = max(0, 22 - __clz(range));  // range >> shift < 1024
      __syncthreads();                    // sh.bin and the histogram are written again
    }
  };
  if (k > 0 && k < p.vocab) select(true, static_cast<u64>(k));
  if (!(top_p >= 1.0f)) select(false, 0);

  // Weights summed in index order: the token (relative to the slice) at which
  // the running sum exceeds aim(total), in the CTA that holds it (-1 in the
  // others); *owner is that CTA's rank.
  auto locate = [&](auto weight, auto aim_of, unsigned* owner, u64* total) -> int {
    u64 mine = 0, all = 0;
    for (int i = tid; i < n; i += kClThreads) mine += weight(i);
    block_scan(mine, sh.scan, &all);
    if (tid == 0) sh.total = all;
    cl.sync();
    u64 sum = 0;
    for (unsigned r = 0; r < C; ++r) sum += *peer(cl, &sh.total, r);
    *total = sum;
    const u64 aim = aim_of(sum);
    u64 base = 0;
    *owner = C - 1;
    for (unsigned r = 0; r < C; ++r) {
      const u64 v = *peer(cl, &sh.total, r);
      if (aim < base + v) {
        *owner = r;
        break;
      }
      base += v;
    }
    if (*owner != rank) return -1;
    constexpr int W = kClThreads / 32;
    const int rounds = (n + kClThreads - 1) / kClThreads;
    u64* table = sh.sums;
    for (int j = 0; j < rounds; ++j) {
      const int i = j * kClThreads + tid;
      u64 v = i < n ? weight(i) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) table[j * W + warp] = v;
    }
    __syncthreads();
    const u64 v = tid < rounds * W ? table[tid] : 0;
    const u64 acc = base + block_scan(v, sh.scan, &all);
    if (acc <= aim && aim < acc + v) sh.bin = tid, sh.before = acc;
    __syncthreads();
    const int i = sh.bin / W * kClThreads + sh.bin % W * 32 + lane;
    const u64 w = i < n ? weight(i) : 0;
    u64 inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sh.before + inc > aim);
    return __shfl_sync(0xffffffffu, i, __ffs(past) - 1);
  };

  int last_tie = 0x7fffffff;  // index of the last token that is kept with the cut's key
  unsigned owner;
  u64 total;
  if (partial) {
    const int at = locate([&](int i) -> u64 { return order_key(xs[i]) == cut.key; },
                          [&](u64) -> u64 { return static_cast<u64>(cut.ties - 1); }, &owner, &total);
    if (at >= 0 && tid == 0) sh.index = i0 + at;
    cl.sync();
    last_tie = *peer(cl, &sh.index, owner);
  }
  auto kept = [&](int i) -> u64 {
    const float l = xs[i];
    const uint32_t key = order_key(l);
    if (key < cut.key || (key == cut.key && i0 + i > last_tie)) return 0;
    const float e = logit_weight(l, rs);
    return e >= min_p || l == top ? fixed_weight(e) : 0;
  };
  const float u = p.uniform[row];
  const int token = locate(kept,
                           [&](u64 all) -> u64 {
                             const double f = static_cast<double>(all) * static_cast<double>(u);
                             return f > 0.0 ? min(static_cast<u64>(f), all - 1) : 0;
                           },
                           &owner, &total);
  if (token >= 0 && tid == 0) {
    p.token[row] = i0 + token;
    if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(kept(token)) / static_cast<double>(total));
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

cudaError_t sample_cluster_launch(const SampleParams& p, int num_sms, cudaStream_t st) {
  static bool ready = false;
  cudaError_t e;
  if (!ready) {
    e = cudaFuncSetAttribute(sample_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceMax * 4);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    ready = true;
  }
  // the fewest CTAs that hold a row; for few rows more of them, down to slices of 2048
  int c = 1;
  while (c * kSliceMax < p.vocab) c *= 2;
  while (c < kClusterMax && static_cast<int64_t>(p.rows) * c * 2 <= num_sms && p.vocab / (2 * c) >= 2048) c *= 2;
  const int slice = ((p.vocab + c - 1) / c + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * static_cast<unsigned>(c));
  cfg.blockDim = dim3(kClThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(slice) * sizeof(float);
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
  if (vocab <= static_cast<uint64_t>(kClusterMax) * kSliceMax) {
    const cudaError_t e = sample_cluster_launch(p, ctx->num_sms, st);
    if (e != cudaSuccess) return check_cuda(ctx, e, "sample");
  } else {
    sample_row_kernel<<<static_cast<unsigned>(rows), kSampleThreads, 0, st>>>(p);
  }
  if (!stream) return finish_op(ctx, "sample");
  return check_cuda(ctx, cudaGetLastError(), "sample");
}
