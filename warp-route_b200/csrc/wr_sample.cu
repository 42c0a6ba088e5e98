// wr_sample.cu — one token for each row of logits, by temperature, top-k,
// top-p and min-p, from a given uniform number.
//
//   w_i = e^((x_i - max) / temperature);   order: x descending, index ascending
//   kept: the first top_k of the order; of these the ones whose preceding sum
//         of w is below top_p times the sum of the first top_k; of these the
//         ones with w_i >= min_p; always the first
//   id  = lowest index whose running sum of kept w, by index, exceeds
//         uniform * sum of kept w
//
// Which token it is hangs on sums passing borders, so w is computed in 64
// bits and held as a whole number of 2^-45: sums of whole numbers do not
// depend on their order, whatever order atomics come in.
//
// A row belongs to one cluster of 1 to 8 CTAs, which reads it once and keeps
// it in shared memory.  The border of the first k, and that of the mass top_p,
// are found without sorting: a histogram (count and mass) of the values over
// 2048 bins, even over [min, max] of the row, tells which bin the border lies
// in; the keys (order-preserving integers) of that bin are binned again until
// one value is left, and equal values go by index.  A few passes over
// shared memory, each followed by an exchange of 2048 sums through distributed
// shared memory; HBM is read once.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <utility>

#include "wr_common.cuh"
#include "wr_internal.h"

namespace cg = cooperative_groups;

namespace wr {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
// 16 vectors a thread hold kSampleMaxVocab values.
constexpr int kMaxSmem = 16 * (kThreads * 16 + kWarps * 8);
constexpr double kMassOne = 35184372088832.0;  // 2^45: with up to 2^18 values sums stay below 2^63
constexpr float kNegInf = -__builtin_huge_valf();

struct SampleArgs {
  const void* logits;
  int64_t row_stride;  // elements
  int vocab;
  int levels;          // vectors of four a thread
  int vec;             // rows allow 16-byte loads
  const float* uniforms;
  const float *temperature, *top_p, *min_p;  // [rows] or null: the numbers below
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;
  int32_t top_k1;
  int64_t* ids;
};

// Order-preserving key of a float that is not NaN.
WR_DEVINL uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

struct Shared {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t warp64[kWarps];
  uint64_t warp64b[kWarps];
  // written by every rank of the cluster into every rank's copy
  uint64_t all_a[2][kMaxCluster], all_b[2][kMaxCluster], all_c[2][kMaxCluster];
  uint64_t found[4];
};

struct Row {
  float max;
  double inv_t;
};
// Weight and its whole number.  Below e^-60 nothing rounds to 2^-45.
WR_DEVINL double weight(const Row& r, float x) {
  if (x == r.max) return 1.0;  // +inf among them
  const double d = ((double)x - (double)r.max) * r.inv_t;
  return d < -60.0 ? 0.0 : exp(d);
}
WR_DEVINL uint64_t mass_of(double w) { return (uint64_t)__double2ll_rn(w * kMassOne); }

// This CTA's part of the row in shared memory: vector l of thread t holds the
// values 4 * ((rank * levels + l) * kThreads + t) .. + 3 of the row, -inf
// behind its end.  A thread touches its own vectors only.
struct Slice {
  float4* v;
  int levels, rank;
  WR_DEVINL int index(int l) const { return ((rank * levels + l) * kThreads + (int)threadIdx.x) * 4; }
  template <typename F>
  WR_DEVINL void each(F f) const {
#pragma unroll 1
    for (int l = 0; l < levels; ++l) {
      const float4 q = v[l * kThreads + threadIdx.x];
      const int i = index(l);
      f(q.x, i);
      f(q.y, i + 1);
      f(q.z, i + 2);
      f(q.w, i + 3);
    }
  }
};

template <typename F>
WR_DEVINL uint64_t warp_reduce(uint64_t v, F f) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Two values of the CTA's threads reduced over the cluster (fa, fb
// associative and commutative); every thread gets both.  `par` alternates
// between calls, so that one call's exchange never meets the next one's.
template <typename FA, typename FB>
WR_DEVINL void cluster_reduce(cg::cluster_group& cl, Shared& s, int& par, uint64_t& a, uint64_t& b,
                              FA fa, FB fb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  a = warp_reduce(a, fa);
  b = warp_reduce(b, fb);
  if (lane == 0) {
    s.warp64[warp] = a;
    s.warp64b[warp] = b;
  }
  __syncthreads();
  const int n = (int)cl.num_blocks(), me = (int)cl.block_rank();
  if (warp == 0) {
    a = s.warp64[lane % kWarps];
    b = s.warp64b[lane % kWarps];
#pragma unroll
    for (int d = 1; d < kWarps; d <<= 1) {
      a = fa(a, __shfl_xor_sync(0xffffffffu, a, d));
      b = fb(b, __shfl_xor_sync(0xffffffffu, b, d));
    }
    if (lane < n) {
      Shared* o = cl.map_shared_rank(&s, lane);
      o->all_a[par][me] = a;
      o->all_b[par][me] = b;
    }
  }
  cl.sync();
  a = s.all_a[par][0];
  b = s.all_b[par][0];
  for (int i = 1; i < n; ++i) {
    a = fa(a, s.all_a[par][i]);
    b = fb(b, s.all_b[par][i]);
  }
  par ^= 1;
}

struct Add { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x + y; } };
struct Max { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x > y ? x : y; } };
struct Min { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x < y ? x : y; } };

// Where the kept part of the order ends: values with key > `key` are kept,
// those equal to it up to and with index `last`.
struct Cut {
  uint32_t key;
  int last;
};
WR_DEVINL bool in_cut(const Cut& c, uint32_t key, int idx) {
  return key > c.key || (key == c.key && idx <= c.last);
}

// The last value of the order (within `within`) whose preceding sum is below
// `target`: sums of 1 (kMass false) or of mass.  kMass: target is top_p times
// the whole mass, of which the first histogram gives the whole.
template <bool kMass>
__device__ __noinline__ Cut find_cut(cg::cluster_group& cl, Shared& s, int& par, const Slice& x,
                                     const Row& row, const Cut& within, uint32_t lo, uint32_t hi,
                                     float low, uint64_t target, float top_p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = (int)cl.num_blocks(), me = (int)cl.block_rank();
  const int seg = kBins / n;  // bins whose sums this rank adds up
  uint64_t above = 0;
  // Even bins over the values first (monotone in x, whatever it rounds to).
  float scale = (float)kBins / (row.max - low);
  bool by_value = scale < 3e38f && scale > 0.f;  // false: max == low or an infinity between them
  for (;;) {
    if (lo == hi) break;
    int shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
    auto bin_of = [&](float v, uint32_t k) {
      if (by_value) return min(kBins - 1, (int)((row.max - v) * scale));
      return (int)((hi - k) >> shift);
    };
    for (int i = tid; i < kBins; i += kThreads) {
      if (kMass) s.mass[i] = 0; else s.count[i] = 0;
    }
    __syncthreads();
    x.each([&](float f, int i) {
      const uint32_t k = key_of(f);
      if (k < lo || k > hi || !in_cut(within, k, i)) return;
      if (kMass) {
        const uint64_t m = mass_of(weight(row, f));
        if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin_of(f, k)]),
                         (unsigned long long)m);
      } else {
        atomicAdd(&s.count[bin_of(f, k)], 1u);
      }
    });
    cl.sync();
    // This rank's bins, summed over the ranks: thread t has bins t * per ...
    // of the segment (seg >= 256, kThreads 512: one to four bins a thread).
    const int per = (seg + kThreads - 1) / kThreads;
    uint64_t v[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = 0;
      const int i = tid * per + e;
      if (e < per && i < seg)
        for (int r = 0; r < n; ++r) {
          const Shared* o = cl.map_shared_rank(&s, r);
          v[e] += kMass ? o->mass[me * seg + i] : (uint64_t)o->count[me * seg + i];
        }
      mine += v[e];
    }
    uint64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint64_t u = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += u;
    }
    if (lane == 31) s.warp64[warp] = incl;
    __syncthreads();
    uint64_t before = incl - mine, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s.warp64[w];
      total += s.warp64[w];
    }
    if (tid < n) cl.map_shared_rank(&s, tid)->all_a[par][me] = total;
    cl.sync();
    uint64_t whole = 0, start = above;
    for (int r = 0; r < n; ++r) {
      whole += s.all_a[par][r];
      if (r < me) start += s.all_a[par][r];
    }
    par ^= 1;
    if (kMass && target == 0) {  // the first histogram: top_p of the whole, rounded up
      const uint64_t p = (uint64_t)((double)top_p * 18446744073709551616.0);
      target = __umul64hi(p, whole) + (p * whole != 0 ? 1 : 0);
      if (target == 0) target = 1;  // top_p 0: the first alone
    }
    // The last bin with something in it whose preceding sum is below target.
    before += start;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < per && v[e] && before < target && before + v[e] >= target) {
        const int bin = me * seg + tid * per + e;
        for (int r = 0; r < n; ++r) {
          Shared* o = cl.map_shared_rank(&s, r);
          o->found[0] = (uint64_t)bin;
          o->found[1] = before;
        }
      }
      before += v[e];
    }
    cl.sync();
    const int bin = (int)s.found[0];
    above = s.found[1];
    // The keys of that bin.
    uint64_t a = 0xffffffffull, b = 0;
    x.each([&](float f, int i) {
      const uint32_t k = key_of(f);
      if (k < lo || k > hi || !in_cut(within, k, i) || bin_of(f, k) != bin) return;
      if (kMass && mass_of(weight(row, f)) == 0) return;
      a = min(a, (uint64_t)k);
      b = max(b, (uint64_t)k);
    });
    cluster_reduce(cl, s, par, a, b, Min(), Max());
    lo = (uint32_t)a;
    hi = (uint32_t)b;
    by_value = false;
  }
  // Equal values: the first r by index.  Each counts one, or its mass.
  Cut c;
  c.key = lo;
  uint64_t each = 1;
  if (kMass) {
    const uint32_t u = lo & 0x80000000u ? lo ^ 0x80000000u : ~lo;
    each = mass_of(weight(row, __uint_as_float(u)));
  }
  if (kMass && target == 0) {  // all values equal: no histogram was made
    uint64_t cnt = 0, none = 0;
    x.each([&](float f, int i) { cnt += key_of(f) == lo && in_cut(within, lo, i); });
    cluster_reduce(cl, s, par, cnt, none, Add(), Add());
    const uint64_t whole = cnt * each, p = (uint64_t)((double)top_p * 18446744073709551616.0);
    target = __umul64hi(p, whole) + (p * whole != 0 ? 1 : 0);
    if (target == 0) target = 1;
  }
  const uint64_t r = each ? (target - above + each - 1) / each : 1;
  uint64_t cnt = 0, none = 0;
  x.each([&](float f, int i) { cnt += key_of(f) == lo && in_cut(within, lo, i); });
  cluster_reduce(cl, s, par, cnt, none, Add(), Add());
  if (r >= cnt) {
    c.last = 0x7fffffff;
    return c;
  }
  // Bisection over the index: rare (ties across the border), at most 18 steps.
  int a = 0, b = 1 << 18;  // ties with index < a: fewer than r; with index < b: at least r
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    uint64_t q = 0;
    none = 0;
    x.each([&](float f, int i) { q += key_of(f) == lo && i < mid && in_cut(within, lo, i); });
    cluster_reduce(cl, s, par, q, none, Add(), Add());
    if (q >= r) b = mid; else a = mid;
  }
  c.last = b - 1;
  return c;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) float4 s_values[];
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  auto started = cl.barrier_arrive();  // a rank's memory is there once it runs
  const int n = (int)cl.num_blocks(), me = (int)cl.block_rank();
  const int64_t r = blockIdx.x / n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* p = static_cast<const T*>(a.logits) + r * a.row_stride;
  const Slice x{s_values, a.levels, me};
  uint64_t* s_level = reinterpret_cast<uint64_t*>(s_values + a.levels * kThreads);  // [levels][kWarps]
  // Maximum with its lowest index, and the lowest value above -inf.
  uint64_t best = 0, low = ~0ull;
#pragma unroll 4
  for (int l = 0; l < a.levels; ++l) {
    const int j = x.index(l);
    float f[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
    if (a.vec && j + 3 < a.vocab) {
      if constexpr (sizeof(T) == 4) {
        const uint4 v = ldg_nc_v4(p + j);
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + j));
        f[0] = bf16lo(v.x); f[1] = bf16hi(v.x);
        f[2] = bf16lo(v.y); f[3] = bf16hi(v.y);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < a.vocab) f[e] = load_scalar<T>(p, j + e);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // NaN counts as -inf; -0 as 0 (equal numbers have equal keys).
      f[e] = f[e] != f[e] ? kNegInf : f[e] + 0.f;
      const uint32_t k = key_of(f[e]);
      best = max(best, ((uint64_t)k << 32) | (0x7fffffffu - (uint32_t)(j + e)));
      if (f[e] > kNegInf) low = min(low, (uint64_t)k);
    }
    s_values[l * kThreads + tid] = make_float4(f[0], f[1], f[2], f[3]);
  }

  const float temp = a.temperature ? a.temperature[r] : a.temperature1;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p1;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p1;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k1;

  int par = 0;
  cl.barrier_wait(std::move(started));
  cluster_reduce(cl, s, par, best, low, Max(), Min());
  const uint32_t kmax = (uint32_t)(best >> 32);
  const int imax = (int)(0x7fffffffu - (uint32_t)best);
  if (low == ~0ull || !(temp > 0.f)) {  // nothing to sample, or the maximum itself
    if (me == 0 && tid == 0) a.ids[r] = low == ~0ull ? -1 : imax;
    return;
  }
  Row row;
  row.max = __uint_as_float(kmax & 0x80000000u ? kmax ^ 0x80000000u : ~kmax);
  row.inv_t = 1.0 / (double)temp;
  const uint32_t klow = (uint32_t)low;
  const float lowest = __uint_as_float(klow & 0x80000000u ? klow ^ 0x80000000u : ~klow);

  Cut cut{0u, 0x7fffffff};  // everything
  if (top_k >= 1 && top_k < a.vocab) {
    // fewer finite values than top_k: nothing is cut
    uint64_t cnt = 0, none = 0;
    x.each([&](float f, int) { cnt += f > kNegInf; });
    cluster_reduce(cl, s, par, cnt, none, Add(), Add());
    if ((uint64_t)top_k < cnt)
      cut = find_cut<false>(cl, s, par, x, row, cut, klow, kmax, lowest, (uint64_t)top_k, 0.f);
  }
  if (top_p < 1.f) {
    const uint32_t from = max(cut.key, klow);
    const float fl = __uint_as_float(from & 0x80000000u ? from ^ 0x80000000u : ~from);
    cut = find_cut<true>(cl, s, par, x, row, cut, from, kmax, fl, 0, fmaxf(top_p, 0.f));
  }

  // Running sums by index: (rank, level, warp, lane, element).
  const Cut keep = cut;
  auto kept_mass = [&](float f, int i) -> uint64_t {
    if (!(f > kNegInf) || !in_cut(keep, key_of(f), i)) return 0;
    const double w = weight(row, f);
    return w >= (double)min_p || i == imax ? mass_of(w) : 0;
  };
  auto level_mass = [&](int l) -> uint64_t {
    const float4 q = s_values[l * kThreads + tid];
    const int i = x.index(l);
    return kept_mass(q.x, i) + kept_mass(q.y, i + 1) + kept_mass(q.z, i + 2) + kept_mass(q.w, i + 3);
  };
  uint64_t sum = 0;
#pragma unroll 1
  for (int l = 0; l < a.levels; ++l) {
    const uint64_t m = level_mass(l), t = warp_reduce(m, Add());
    if (lane == 0) s_level[l * kWarps + warp] = t;
    sum += m;
  }
  // every rank's sum, by rank
  {
    uint64_t t = warp_reduce(sum, Add());
    if (lane == 0) s.warp64[warp] = t;
    __syncthreads();
    if (tid < n) {
      t = 0;
      for (int w = 0; w < kWarps; ++w) t += s.warp64[w];
      cl.map_shared_rank(&s, tid)->all_c[0][me] = t;
    }
    cl.sync();
  }
  uint64_t whole = 0, start = 0;
  for (int i = 0; i < n; ++i) {
    if (i < me) start += s.all_c[0][i];
    whole += s.all_c[0][i];
  }
  const uint64_t here = s.all_c[0][me];
  const double u = fmin(fmax((double)a.uniforms[r], 0.0), 1.0 - 1.0 / 16777216.0);
  const uint64_t goal = __umul64hi((uint64_t)(u * 18446744073709551616.0), whole);  // < whole
  if (goal < start || goal >= start + here) return;
  uint64_t at = start;
  int l = 0, w0 = 0;
  for (int i = 0; i < a.levels * kWarps; ++i) {  // the (level, warp) that passes the goal
    const uint64_t t = s_level[i];
    if (goal < at + t) {
      l = i / kWarps;
      w0 = i % kWarps;
      break;
    }
    at += t;
  }
  if (warp != w0) return;
  const uint64_t m = level_mass(l);
  uint64_t incl = m;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  at += incl - m;
  if (goal < at || goal >= at + m) return;
  const float4 q = s_values[l * kThreads + tid];
  const float f[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t t = kept_mass(f[e], x.index(l) + e);
    if (goal >= at && goal < at + t) a.ids[r] = x.index(l) + e;
    at += t;
  }
}

template <typename T>
cudaError_t launch_rows(const SampleArgs& a, int64_t rows, int cluster, cudaStream_t stream) {
  const void* k = reinterpret_cast<const void*>(k_sample<T>);
  const int smem = a.levels * (kThreads * 16 + kWarps * 8);
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  void* args[1] = {const_cast<SampleArgs*>(&a)};
  return cudaLaunchKernelExC(&cfg, k, args);
}

}  // namespace

wr_status_t launch_sample(const SampleProblem& p, cudaStream_t stream) {
  SampleArgs a{};
  a.logits = p.logits;
  a.row_stride = p.row_stride;
  a.vocab = p.vocab;
  const int elt = p.dtype == WR_DTYPE_BF16 ? 2 : 4;
  const int need = elt == 4 ? 16 : 8;  // bytes of a vector of four
  a.vec = (reinterpret_cast<uintptr_t>(p.logits) % need) == 0 && (p.row_stride * elt) % need == 0;
  a.uniforms = p.uniforms;
  a.temperature = p.temperatures; a.top_p = p.top_ps; a.min_p = p.min_ps; a.top_k = p.top_ks;
  a.temperature1 = p.temperature; a.top_p1 = p.top_p; a.min_p1 = p.min_p; a.top_k1 = p.top_k;
  a.ids = p.ids;
  // The smallest cluster whose CTAs hold the row with 8 vectors a thread (64
  // KB, so that two share an SM; fewer exchanges than with more CTAs); with
  // few rows, for their latency, one vector a thread or the largest cluster.
  const int64_t vectors = ((int64_t)p.vocab + 3) / 4;
  const int64_t per = p.rows * kMaxCluster <= device_sm_count() ? kThreads : 8 * kThreads;
  int cluster = 1;
  while (cluster < kMaxCluster && vectors > cluster * per) cluster *= 2;
  a.levels = (int)((vectors + (int64_t)cluster * kThreads - 1) / ((int64_t)cluster * kThreads));
  const cudaError_t e = elt == 2 ? launch_rows<uint16_t>(a, p.rows, cluster, stream)
                                 : launch_rows<float>(a, p.rows, cluster, stream);
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "sample_tokens launch");
}

}  // namespace wr
