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

#include "kib_ctx.cuh"

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
KIB_DEV u64 fixed_weight(float e) { return static_cast<u64>(e * 1099511627776.0f); }

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

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleParams p) {
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

}  // namespace
}  // namespace kib

using namespace kib;

extern "C" int kib_sample_f32(kib_ctx* ctx, const float* logits, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                              const float* uniform, const float* temperature, const int32_t* top_k, const float* top_p,
                              const float* min_p, int32_t* token_out, float* prob_out, void* stream) {
  KIB_REQUIRE_CTX(ctx);
  KIB_ARG(vocab > 0 && vocab <= (1ull << 23), "sample: vocab must be in 1..2^23");
  KIB_ARG(rows < (1ull << 31), "sample: rows out of range");
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
  sample_kernel<<<static_cast<unsigned>(rows), kSampleThreads, 0, stream ? static_cast<cudaStream_t>(stream) : ctx->stream>>>(p);
  if (!stream) return finish_op(ctx, "sample");
  return check_cuda(ctx, cudaGetLastError(), "sample");
}
