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
// A row belongs to one cluster of 1 to 8 CTAs: as many as run at once for all
// rows (two an SM), and enough to keep the row in shared memory with two CTAs
// an SM (256 rows of 131072: 8 CTAs a row 214 us, one that reads the row again
// for each pass 345 us); only what 8 CTAs do not hold is read again for each
// pass, from L2 as a rule.  The border of the first k, and that of the mass
// top_p, are found without sorting the row: a histogram of the values over
// 1024 bins, even over [min, max] of the row, tells which bin a border lies
// in, for the first k exactly, for the mass by count times weight of the mean of
// a bin, after which one pass over the exact weights says which of the three
// bins around it it is (no atomics on masses: they took longer than the
// weights).  That bin's values, few as a rule, are gathered by one CTA, sorted
// and cut exactly; with a short top_k everything down to its border goes there,
// and that CTA ends the row.  A bin with more values than fit there (rows of
// many equal values) is binned again by key until one value is left.  What
// bounds the kernel is the chain of passes and exchanges for few rows and the
// 64-bit arithmetic of the weights for many.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "wr_common.cuh"
#include "wr_internal.h"

namespace cg = cooperative_groups;

namespace wr {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kMaxCluster = 8;
constexpr int kList = 1024;  // values that one CTA sorts
constexpr int kTable = 128;  // steps of the exponential's table per factor of two
constexpr int kKeepBytes = 76 * 1024;  // of a row's part in shared memory, at most
constexpr int kFlight = 4;             // vectors a thread has in flight
constexpr double kMassOne = 35184372088832.0;  // 2^45: with up to 2^18 values sums stay below 2^63
constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
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

// Order-preserving key of a float that is not NaN, and back.
WR_DEVINL uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
WR_DEVINL float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Where the kept part of the order ends: values with key > `key` are kept,
// those equal to it up to and with index `last`.
struct Cut {
  uint32_t key;
  int last;
};
WR_DEVINL bool in_cut(const Cut& c, uint32_t key, int idx) {
  return key > c.key || (key == c.key && idx <= c.last);
}

struct alignas(16) Shared {
  uint32_t count[kBins];
  // Masses in parts of 14 bits, each added with a native 32-bit atomic (a
  // 64-bit one is a loop of compare and swap): at most 2^18 values, so no part
  // passes 32 bits.
  uint32_t mass[4][kBins];
  uint64_t list[kList];  // (key, ~index); rank 0's alone is used
  double table[kTable];
  uint64_t warp64[kWarps];
  uint64_t warp64b[kWarps];
  // written by every rank of the cluster into every rank's copy
  uint64_t all_a[2][kMaxCluster], all_b[2][kMaxCluster];
  uint64_t all_w[kMaxCluster][5];
  uint64_t warp_w[kWarps][5];
  uint32_t rank[256];
  uint64_t found[2][4];
  uint32_t listed;
};

WR_DEVINL void add_mass(Shared& s, int bin, uint64_t m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t part = (uint32_t)(m >> (14 * i)) & 0x3fffu;
    if (part) atomicAdd(&s.mass[i][bin], part);
  }
}
static_assert(kSampleMaxVocab <= 1 << 18, "parts of the masses");
WR_DEVINL void clear_bins(Shared& s) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) s.mass[j][i] = 0;
  }
}

static_assert(sizeof(Shared) % 16 == 0 && sizeof(Shared) + kKeepBytes < 113 * 1024, "two CTAs an SM");

struct Row {
  float max;
  float low;            // values below this weigh nothing: their weight rounds to 0, or they are -inf
  double maxd;
  double steps;         // table steps per unit of x: kTable * log2(e) / temperature
  const double* table;  // 2^(i / kTable)
};

// The same value in 64 bits, by its bits (the conversion is one of the slow
// instructions).  A number below 2^-126 in size comes out as some other one
// below 2^-126, an infinity as 2^128: no difference to x - max where it counts.
WR_DEVINL double wider(float x) {
  const uint32_t b = __float_as_uint(x);
  return __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)), (int)(b << 29));
}

// w = 2^(steps (x - max) / kTable): the whole steps by the table and the
// exponent, the rest r of at most half a step by the series of the exponential
// of u = r ln 2 / kTable (|u| <= ln 2 / 256) up to u^4 (the next term is below
// 2^-49).  Table-driven reduction as in P. T. P. Tang, ACM TOMS 15 (1989).
WR_DEVINL double weight(const Row& r, float x) {
  if (!(x >= r.low)) return 0.0;
  constexpr double c = 0.69314718055994530942 / kTable;
  const double t = (wider(x) - r.maxd) * r.steps;
  const double m = t + kMagic;
  const int k = __double2loint(m);
  const double u = t - (m - kMagic);
  const double e = fma(fma(fma(fma(u, c * c * c * c / 24, c * c * c / 6), u, c * c / 2), u, c), u, 1.0);
  const double w = r.table[k & (kTable - 1)] * e;
  return __hiloint2double(__double2hiint(w) + ((k >> 7) << 20), __double2loint(w));
}
static_assert(kTable == 128, "the shift above");
// Rounded to a whole number of 2^-45 (w <= 1).
WR_DEVINL uint64_t mass_of(double w) {
  return (uint64_t)__double_as_longlong(fma(w, kMassOne, 4503599627370496.0)) & 0xfffffffffffffull;
}

// This CTA's part of the row: vector l of thread t is the four values from
// 4 * ((rank * levels + l) * kThreads + t) on, -inf behind the row's end, NaN
// as -inf and -0 as 0 (equal numbers have equal keys).  kKeep: in shared
// memory, as they came (float4 or uint2), where a thread touches its own
// vectors only; else they are read from the row each time.
template <typename T>
struct Four;
template <>
struct Four<float> { using V = float4; };
template <>
struct Four<uint16_t> { using V = uint2; };
WR_DEVINL void widen4(const float4& v, float (&f)[4]) { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
WR_DEVINL void widen4(const uint2& v, float (&f)[4]) {
  f[0] = bf16lo(v.x); f[1] = bf16hi(v.x);
  f[2] = bf16lo(v.y); f[3] = bf16hi(v.y);
}
WR_DEVINL void pack4(const float (&f)[4], float4& v) { v = make_float4(f[0], f[1], f[2], f[3]); }
WR_DEVINL void pack4(const float (&f)[4], uint2& v) {  // exact: they came from bf16
  v.x = (__float_as_uint(f[0]) >> 16) | (__float_as_uint(f[1]) & 0xffff0000u);
  v.y = (__float_as_uint(f[2]) >> 16) | (__float_as_uint(f[3]) & 0xffff0000u);
}
template <typename T, bool kKeep>
struct Slice {
  using V = typename Four<T>::V;
  V* kept;
  const T* row;
  int levels, rank, vocab;
  bool vec;
  WR_DEVINL int index(int l) const { return ((rank * levels + l) * kThreads + (int)threadIdx.x) * 4; }
  WR_DEVINL V fetch(int l) const {  // from the row
    const int j = index(l);
    if (vec && j + 3 < vocab) return __ldg(reinterpret_cast<const V*>(row + j));
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = j + e < vocab ? load_scalar<T>(row, j + e) : kNegInf;
    V v;
    pack4(f, v);
    return v;
  }
  static WR_DEVINL void clean(float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = f[e] != f[e] ? kNegInf : f[e] + 0.f;
  }
  WR_DEVINL void four(int l, float (&f)[4]) const {
    widen4(kKeep ? kept[l * kThreads + threadIdx.x] : fetch(l), f);
    if (!kKeep) clean(f);
  }
  // f(value, index) for each value; kStore: reads the row and keeps it.
  template <bool kStore = false, typename F>
  WR_DEVINL void each(F f) const {
    constexpr bool kRead = !kKeep || kStore;
    constexpr int U = kRead ? kFlight : 1;
#pragma unroll 1
    for (int l0 = 0; l0 < levels; l0 += U) {
      V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (l0 + u < levels) v[u] = kRead ? fetch(l0 + u) : kept[(l0 + u) * kThreads + threadIdx.x];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (l0 + u >= levels) continue;
        float q[4];
        widen4(v[u], q);
        if (kRead) clean(q);
        if (kKeep && kStore) pack4(q, kept[(l0 + u) * kThreads + threadIdx.x]);
        const int i = index(l0 + u);
#pragma unroll
        for (int e = 0; e < 4; ++e) f(q[e], i + e);
      }
    }
  }
};

struct Add { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x + y; } };
struct Max { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x > y ? x : y; } };
struct Min { WR_DEVINL uint64_t operator()(uint64_t x, uint64_t y) const { return x < y ? x : y; } };

template <typename F>
WR_DEVINL uint64_t warp_reduce(uint64_t v, F f) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
WR_DEVINL uint64_t warp_inclusive(uint64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += u;
  }
  return v;
}

WR_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
WR_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The cluster and what its exchanges go through.  Each exchange writes into
// the copy of all_* or found that `par` names and flips it: a rank can write
// into a copy again only after a cluster barrier that every rank reaches after
// reading it.
struct Group {
  cg::cluster_group cl;
  Shared* s;
  int n, me, par;

  WR_DEVINL void sync() {
    if (n == 1) __syncthreads(); else cl.sync();
  }
  WR_DEVINL Shared* of(int rank) { return n == 1 ? s : cl.map_shared_rank(s, rank); }

  // A value for rank 0's list, from the lanes that have one (one atomic a
  // warp); all lanes of the warp call it.
  WR_DEVINL void push(bool have, float f, int i) {
    const uint32_t who = __ballot_sync(0xffffffffu, have);
    if (!who) return;
    const int lane = threadIdx.x & 31, first = __ffs(who) - 1;
    Shared* o = of(0);
    uint32_t at = 0;
    if (lane == first) at = atomicAdd(&o->listed, (uint32_t)__popc(who));
    at = __shfl_sync(0xffffffffu, at, first) + __popc(who & ((1u << lane) - 1));
    if (have && at < (uint32_t)kList) o->list[at] = ((uint64_t)key_of(f) << 32) | (uint32_t)~i;
  }

  // Two values of the CTA's threads reduced over the cluster (fa, fb
  // associative and commutative); every thread gets both.
  template <typename FA, typename FB>
  WR_DEVINL void reduce(uint64_t& a, uint64_t& b, FA fa, FB fb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    a = warp_reduce(a, fa);
    b = warp_reduce(b, fb);
    if (lane == 0) {
      s->warp64[warp] = a;
      s->warp64b[warp] = b;
    }
    __syncthreads();
    if (warp == 0) {
      a = s->warp64[lane % kWarps];
      b = s->warp64b[lane % kWarps];
#pragma unroll
      for (int d = 1; d < kWarps; d <<= 1) {
        a = fa(a, __shfl_xor_sync(0xffffffffu, a, d));
        b = fb(b, __shfl_xor_sync(0xffffffffu, b, d));
      }
      if (lane < n) {
        Shared* o = of(lane);
        o->all_a[par][me] = a;
        o->all_b[par][me] = b;
      }
    }
    sync();
    a = s->all_a[par][0];
    b = s->all_b[par][0];
    for (int i = 1; i < n; ++i) {
      a = fa(a, s->all_a[par][i]);
      b = fb(b, s->all_b[par][i]);
    }
    par ^= 1;
  }

  // Five sums over the cluster.
  WR_DEVINL void reduce5(uint64_t (&v)[5]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      v[i] = warp_reduce(v[i], Add());
      if (lane == 0) s->warp_w[warp][i] = v[i];
    }
    __syncthreads();
    if (threadIdx.x < 5 * n) {
      const int i = threadIdx.x % 5;
      uint64_t t = 0;
      for (int w = 0; w < kWarps; ++w) t += s->warp_w[w][i];
      of(threadIdx.x / 5)->all_w[me][i] = t;
    }
    sync();
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      v[i] = 0;
      for (int r = 0; r < n; ++r) v[i] += s->all_w[r][i];
    }
  }

  // This rank's share of the bins, kBins / n of them from first_bin(), one to
  // four a thread, summed over the ranks; and what lies before a thread's
  // first one in the whole order, and in all of it.
  struct Bins {
    uint64_t v[4], before, whole;
  };
  WR_DEVINL int share() const { return kBins / n; }
  WR_DEVINL int per() const { return (share() + kThreads - 1) / kThreads; }
  WR_DEVINL int first_bin() const { return me * share() + (int)threadIdx.x * per(); }

  // After the histograms are whole (a cluster barrier).  Both sums at once:
  // counts and masses (kMass), or counts and what of_bin makes of a bin, its
  // count and its values' summed places inside it (kept in mass[0]).
  template <bool kMass, typename F>
  WR_DEVINL void sum_bins(Bins& c, Bins& m, F of_bin) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t sc = 0, sm = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c.v[e] = m.v[e] = 0;
      if (e < per() && (int)threadIdx.x * per() + e < share()) {
        const int b = first_bin() + e;
        if constexpr (kMass) {
          for (int r = 0; r < n; ++r) {
            const Shared* o = of(r);
            for (int i = 0; i < 4; ++i) m.v[e] += (uint64_t)o->mass[i][b] << (14 * i);
          }
        } else {
          uint32_t offsets = 0;
          if (n == 1) {
            c.v[e] = s->count[b];
            offsets = s->mass[0][b];
          } else {
            uint32_t x[kMaxCluster], y[kMaxCluster];  // all at once: each takes some thousand cycles
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
              const Shared* o = of(r < n ? r : 0);
              x[r] = o->count[b];
              y[r] = o->mass[0][b];
            }
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
              c.v[e] += r < n ? x[r] : 0;
              offsets += r < n ? y[r] : 0;
            }
          }
          m.v[e] = c.v[e] ? of_bin(b, (float)c.v[e], (float)offsets) : 0;
        }
      }
      sc += c.v[e];
      sm += m.v[e];
    }
    const uint64_t ic = warp_inclusive(sc, lane), im = warp_inclusive(sm, lane);
    if (lane == 31) {
      s->warp64[warp] = ic;
      s->warp64b[warp] = im;
    }
    __syncthreads();
    c.before = ic - sc;
    m.before = im - sm;
    uint64_t tc = 0, tm = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        c.before += s->warp64[w];
        m.before += s->warp64b[w];
      }
      tc += s->warp64[w];
      tm += s->warp64b[w];
    }
    if ((int)threadIdx.x < n) {
      Shared* o = of(threadIdx.x);
      o->all_a[par][me] = tc;
      o->all_b[par][me] = tm;
    }
    sync();
    c.whole = m.whole = 0;
    for (int r = 0; r < n; ++r) {
      if (r < me) {
        c.before += s->all_a[par][r];
        m.before += s->all_b[par][r];
      }
      c.whole += s->all_a[par][r];
      m.whole += s->all_b[par][r];
    }
    par ^= 1;
  }

  // The last bin with something of x in it whose preceding sum is below
  // target (0 < target <= x.whole); the sums of x and y before it, and that of
  // x up to its end.
  WR_DEVINL int find_bin(const Bins& x, const Bins& y, uint64_t target, uint64_t& bx, uint64_t& by,
                         uint64_t& ex) {
    uint64_t before = x.before, other = y.before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (x.v[e] && before < target && before + x.v[e] >= target)
        for (int r = 0; r < n; ++r) {
          Shared* o = of(r);
          o->found[par][0] = (uint64_t)(first_bin() + e);
          o->found[par][1] = before;
          o->found[par][2] = other;
          o->found[par][3] = before + x.v[e];
        }
      before += x.v[e];
      other += y.v[e];
    }
    sync();
    const int bin = (int)s->found[par][0];
    bx = s->found[par][1];
    by = s->found[par][2];
    ex = s->found[par][3];
    par ^= 1;
    return bin;
  }
};

// Sorts list[0 .. n) descending (n <= kList), all threads of the CTA.  Up to
// 256 entries by counting the larger ones (entries differ), a few barriers;
// more by a bitonic network.  Entries up to the next power of two become 0 in
// the latter.
__device__ __noinline__ void sort_list(uint64_t* list, uint32_t* rank, int n) {
  if (n <= 256) {
    int size = 32;
    while (size < n) size *= 2;
    const int e = threadIdx.x & (size - 1), part = threadIdx.x / size, parts = kThreads / size;
    if (threadIdx.x < 256) rank[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t mine = e < n ? list[e] : 0;
    uint32_t larger = 0;
    for (int j = part; j < n; j += parts) larger += list[j] > mine;
    if (e < n && larger) atomicAdd(&rank[e], larger);
    __syncthreads();
    if (part == 0 && e < n) list[rank[e]] = mine;
    __syncthreads();
    return;
  }
  int size = 32;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
  for (int k = 2; k <= size; k *= 2)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int lo = ((i & ~(j - 1)) << 1) | (i & (j - 1)), hi = lo | j;
        const uint64_t a = list[lo], b = list[hi];
        if ((a < b) == ((lo & k) == 0)) {
          list[lo] = b;
          list[hi] = a;
        }
      }
    }
  __syncthreads();
}

// top_p (below 1) of a mass, rounded up to a whole number and at least 1: a
// value is kept if the mass before it is below this.
WR_DEVINL uint64_t mass_target(float top_p, uint64_t whole) {
  const uint64_t p = (uint64_t)((double)fmaxf(top_p, 0.f) * 18446744073709551616.0);
  const uint64_t t = __umul64hi(p, whole) + (p * whole != 0 ? 1 : 0);
  return t ? t : 1;
}

// uniform * whole, rounded down (so below whole): the token's running sum
// exceeds it.
WR_DEVINL uint64_t goal_of(float uniform, uint64_t whole) {
  const double u = fmin(fmax((double)uniform, 0.0), 1.0 - 1.0 / 16777216.0);
  return __umul64hi((uint64_t)(u * 18446744073709551616.0), whole);
}

// Exclusive running sum over the CTA's threads, and the whole.
WR_DEVINL uint64_t cta_before(Shared& s, uint64_t v, uint64_t& whole) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t incl = warp_inclusive(v, lane);
  __syncthreads();
  if (lane == 31) s.warp64[warp] = incl;
  __syncthreads();
  uint64_t before = incl - v;
  whole = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s.warp64[w];
    whole += s.warp64[w];
  }
  return before;
}

// The rest of a row whose first top_k all lie in the list (n >= top_k values
// of it, unsorted): one CTA, two list entries a thread.
__device__ __noinline__ void finish_list(Shared& s, const Row row, int n, int top_k, float top_p,
                                         float min_p, float uniform, int64_t* id) {
  constexpr int kPer = kList / kThreads;
  sort_list(s.list, s.rank, n);
  uint64_t entry[kPer], m[kPer], sum = 0, whole;
  bool keep[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = threadIdx.x * kPer + e;
    keep[e] = i < top_k && i < n;
    entry[e] = keep[e] ? s.list[i] : 0;
    const double w = keep[e] ? weight(row, value_of((uint32_t)(entry[e] >> 32))) : 0.0;
    m[e] = mass_of(w);
    sum += m[e];
    keep[e] = keep[e] && (w >= (double)min_p || i == 0);
  }
  uint64_t before = cta_before(s, sum, whole);
  if (top_p < 1.f) {
    const uint64_t target = mass_target(top_p, whole);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      keep[e] = keep[e] && before < target;
      before += m[e];
    }
  }
  // By index: the kept entries again, as (~index, key).
  uint64_t kept = 0, all;
#pragma unroll
  for (int e = 0; e < kPer; ++e) kept += keep[e];
  int at = (int)cta_before(s, kept, all);
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (keep[e]) s.list[at++] = (entry[e] << 32) | (entry[e] >> 32);
  __syncthreads();
  sort_list(s.list, s.rank, (int)all);
  sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = threadIdx.x * kPer + e;
    entry[e] = i < (int)all ? s.list[i] : 0;
    m[e] = entry[e] ? mass_of(weight(row, value_of((uint32_t)entry[e]))) : 0;
    sum += m[e];
  }
  before = cta_before(s, sum, whole);
  const uint64_t goal = goal_of(uniform, whole);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (goal >= before && goal < before + m[e]) *id = (int64_t)(uint32_t)~(uint32_t)(entry[e] >> 32);
    before += m[e];
  }
}

// A border inside keys [lo, hi] (all of them within `within`), where `above`
// lies before them in the order: the last value whose preceding sum is below
// target, sums of 1 (kMass false) or of mass.  For bins too full to sort:
// binned by key until one key is left, whose values go by index.  Four passes
// of 1024 bins tell any two keys apart.
// (By value, and `par` back by value: nothing of the kernel's hot loops may
// have its address taken, or they would read it from memory each time.)
struct CutPar {
  Cut cut;
  int par;
};
template <bool kMass, typename X>
__device__ __noinline__ CutPar find_by_key(Group g, const X x, const Row row, const Cut within,
                                        uint32_t lo, uint32_t hi, uint64_t above, uint64_t target) {
  Shared& s = *g.s;
  for (int pass = 0; pass < 4 && lo < hi; ++pass) {
    int shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
    clear_bins(s);
    __syncthreads();
    x.each([&](float f, int i) {
      const uint32_t k = key_of(f);
      if (k < lo || k > hi || !in_cut(within, k, i)) return;
      add_mass(s, (int)((hi - k) >> shift), kMass ? mass_of(weight(row, f)) : 1);
    });
    g.sync();
    Group::Bins c, m;
    g.sum_bins<true>(c, m, 0);
    uint64_t before, none, end;
    const int bin = g.find_bin(m, c, target - above, before, none, end);
    above += before;
    uint64_t a = 0xffffffffull, b = 0;
    x.each([&](float f, int i) {
      const uint32_t k = key_of(f);
      if (k < lo || k > hi || (int)((hi - k) >> shift) != bin || !in_cut(within, k, i)) return;
      a = min(a, (uint64_t)k);
      b = max(b, (uint64_t)k);
    });
    g.reduce(a, b, Min(), Max());
    lo = (uint32_t)a;
    hi = (uint32_t)b;
  }
  // Equal values: the first r by index.
  Cut c;
  c.key = lo;
  const uint64_t each = kMass ? mass_of(weight(row, value_of(lo))) : 1;
  const uint64_t r = each ? (target - above + each - 1) / each : 1;
  const int most = lo == within.key ? within.last : 0x7fffffff;
  int a = 0, b = 1 << 18;  // fewer than r of them have an index below a; r or more below b, or b is the end
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    uint64_t q = 0, none = 0;
    x.each([&](float f, int i) { q += key_of(f) == lo && i < mid && i <= most; });
    g.reduce(q, none, Add(), Add());
    if (q >= r) b = mid; else a = mid;
  }
  c.last = min(b - 1, most);
  return CutPar{c, g.par};
}

template <typename T, bool kKeep>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t s_dynamic[];
  Shared& s = *reinterpret_cast<Shared*>(s_dynamic);
  Group g{cg::this_cluster(), &s, 0, 0, 0};
  g.n = (int)g.cl.num_blocks();
  g.me = (int)g.cl.block_rank();
  if (g.n > 1) cluster_arrive();  // a rank's memory is there once it runs
  const int64_t r = blockIdx.x / g.n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* s_level = reinterpret_cast<uint64_t*>(s_dynamic + sizeof(Shared));  // [levels][kWarps]
  const Slice<T, kKeep> x{reinterpret_cast<typename Four<T>::V*>(s_level + a.levels * kWarps),
                          static_cast<const T*>(a.logits) + r * a.row_stride, a.levels, g.me, a.vocab, a.vec != 0};
  // Maximum with its lowest index, and the lowest value above -inf.
  float top = kNegInf, least = __builtin_huge_valf();
  int at_top = 0x7fffffff;
  x.template each<true>([&](float f, int i) {
    if (f > top) {
      top = f;
      at_top = i;
    }
    if (f > kNegInf) least = fminf(least, f);
  });
  uint64_t best = ((uint64_t)key_of(top) << 32) | (0x7fffffffu - (uint32_t)at_top);
  uint64_t low = top > kNegInf ? (uint64_t)key_of(least) : ~0ull;
  if (tid < kTable) s.table[tid] = exp2((double)tid / kTable);
  if (tid == 0) s.listed = 0;
  clear_bins(s);
  const float temp = a.temperature ? a.temperature[r] : a.temperature1;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p1;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p1;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k1;

  if (g.n > 1) cluster_wait();
  g.reduce(best, low, Max(), Min());
  const uint32_t kmax = (uint32_t)(best >> 32), klow = (uint32_t)low;
  const int imax = (int)(0x7fffffffu - (uint32_t)best);
  if (low == ~0ull || !(temp > 0.f)) {  // nothing to sample, or the maximum itself
    if (g.me == 0 && tid == 0) a.ids[r] = low == ~0ull ? -1 : imax;
    return;
  }
  Row row;
  row.max = value_of(kmax);
  row.maxd = wider(row.max);
  // e^-41.6 is 2^-60, far below the 2^-46 that rounds to nothing
  const float lowest = value_of((uint32_t)low);
  row.low = row.max == __builtin_huge_valf() ? row.max : fmaxf(row.max - 41.6f * temp, lowest);
  row.steps = kTable * 1.4426950408889634074 / (double)temp;
  row.table = s.table;

  Cut cut{0u, 0x7fffffff};  // everything
  bool by_k = top_k >= 1 && top_k < a.vocab;
  const bool by_p = top_p < 1.f;
  if (by_k || by_p) {
    // Even bins over the values (monotone in x, whatever it rounds to).  A
    // value's bin is the whole part of its rounded place, in every pass: places
    // are compared with whole numbers only, never shifted and rounded again.
    const float scale = (float)kBins / (row.max - value_of(klow));
    const bool even = scale > 0.f && scale < 3e38f;  // not: one value, or an infinite span
    Group::Bins cnt, mass;  // mass: about, in 2^-30
    const float width = (row.max - value_of(klow)) / kBins;
    auto place = [&](float f) { return __fmul_rn(__fsub_rn(row.max, f), scale); };
    auto about = [&](float b) { return exp2f((float)row.steps / kTable * -b * width) * 1073741824.f; };
    if (even) {
      x.each([&](float f, int) {
        if (!(f >= lowest)) return;
        const float y = place(f);
        const int b = min(kBins - 1, (int)y);
        atomicAdd(&s.count[b], 1u);
        // the place inside the bin in 1/256 (at most 2^18 of them: 26 bits)
        if (by_p) atomicAdd(&s.mass[0][b], (uint32_t)min(255, (int)((y - (float)b) * 256.f)));
      });
      g.sync();
      // The mean place of a bin's values: their mean weight to 1e-5.
      g.sum_bins<false>(cnt, mass, [&](int b, float n, float places) {
        return (uint64_t)(n * about((float)b + (places / n + 0.5f) * (1.f / 256)));
      });
    } else {
      uint64_t c = 0, none = 0;
      x.each([&](float f, int) { c += f > kNegInf; });
      g.reduce(c, none, Add(), Add());
      cnt.whole = c;
    }
    if (by_k && (uint64_t)top_k >= cnt.whole) by_k = false;  // fewer values than that
    auto take = [&](CutPar c) {
      cut = c.cut;
      g.par = c.par;
    };
    int listed = 0;
    double share = 1.0;  // about, of the mass: what top_k leaves
    // Without turning each into a whole number: a place is not negative, so
    // its whole part is below b where it is.
    auto bin_end = [](int b) { return b == kBins - 1 ? 3e38f : (float)(b + 1); };
    auto in_bin = [&](float f, int b) {
      const float y = place(f);
      return y >= (float)b && y < bin_end(b);
    };
    // The values of a bin, sorted, in rank 0's list; how many (on all ranks).
    auto gather = [&](int bin) {
      x.each([&](float f, int i) {
        g.push(in_bin(f, bin) && in_cut(cut, key_of(f), i), f, i);
      });
      g.sync();
      listed = (int)g.of(0)->listed;
      if (g.me == 0 && listed <= kList) sort_list(s.list, s.rank, listed);
    };
    // Keys of a bin, for find_by_key.
    auto keys = [&](int bin, uint32_t& lo, uint32_t& hi) {
      uint64_t l = 0xffffffffull, h = 0;
      x.each([&](float f, int) {
        if (!in_bin(f, bin)) return;
        l = min(l, (uint64_t)key_of(f));
        h = max(h, (uint64_t)key_of(f));
      });
      g.reduce(l, h, Min(), Max());
      lo = (uint32_t)l;
      hi = (uint32_t)h;
    };
    if (by_k && even) {
      uint64_t above = 0, above_mass = 0, end = 0;
      const int bin = g.find_bin(cnt, mass, (uint64_t)top_k, above, above_mass, end);
      if (end <= kList) {  // everything down to the border goes to one CTA, which ends the row
        x.each([&](float f, int i) {
          g.push(place(f) < bin_end(bin), f, i);
        });
        g.sync();
        if (g.me == 0) finish_list(s, row, (int)end, top_k, top_p, min_p, a.uniforms[r], a.ids + r);
        return;
      }
      if (mass.whole) share = fmin(1.0, ((double)above_mass + ((double)top_k - (double)above) * about((float)bin + 0.5f)) / (double)mass.whole);
      gather(bin);
      if (listed <= kList) {
        const int need = top_k - (int)above;  // of the bin
        if (g.me == 0 && tid < g.n) g.of(tid)->found[g.par][0] = s.list[need - 1];
        g.sync();
        cut.key = (uint32_t)(s.found[g.par][0] >> 32);
        cut.last = (int)~(uint32_t)s.found[g.par][0];
        g.par ^= 1;
      } else {
        uint32_t lo, hi;
        keys(bin, lo, hi);
        take(find_by_key<false>(g, x, row, cut, lo, hi, above, (uint64_t)top_k));
      }
    } else if (by_k) {
      take(find_by_key<false>(g, x, row, cut, klow, kmax, 0, (uint64_t)top_k));
    }
    if (by_p) {
      // The bin where the border of top_p lies, about; then the exact masses
      // before and in the three bins around it, and of all.
      const Cut within = cut;
      int bin = -1;
      uint64_t target = 0, above = 0;
      bool exact = false;
      uint64_t w[5] = {0, 0, 0, 0, 0};  // all, before the window, its three bins
      if (even && mass.whole) {
        uint64_t none1, none2, none3;
        const uint64_t goal = (uint64_t)((double)mass.whole * share * (double)fmaxf(top_p, 0.f));
        bin = g.find_bin(mass, cnt, min(mass.whole, goal + 1), none1, none2, none3) - 1;
      }
      const float low_f = fmaxf(within.key ? value_of(within.key) : kNegInf, row.low);
      const float cut_f = within.key ? value_of(within.key) : kNegInf;
      const float y0 = even ? (float)bin : -1.f, y3 = even ? y0 + 3.f : -1.f;
      const float y1 = y0 + 1.f, y2 = y0 + 2.f;  // (bin -1 is empty)
      x.each([&](float f, int i) {
        if (!(f >= low_f) || (f == cut_f && i > within.last)) return;
        const uint64_t m = mass_of(weight(row, f));
        w[0] += m;
        const float y = place(f);
        if (y < y0) w[1] += m;
        else if (y < y3) {  // few (in registers: hundreds of 64-bit atomics on three words took longer than the pass)
          if (y < y1) w[2] += m;
          else if (y < y2) w[3] += m;
          else w[4] += m;
        }
      });
      g.reduce5(w);
      target = mass_target(top_p, w[0]);
      above = w[1];
#pragma unroll
      for (int i = 2; i < 5; ++i) {
        if (exact) continue;
        if (even && above < target && above + w[i] >= target) {
          exact = true;
          bin += i - 2;
        } else {
          above += w[i];
        }
      }
      if (exact) {
        if (g.me == 0 && tid == 0) s.listed = 0;
        g.sync();
        gather(bin);
      }
      if (exact && listed <= kList) {
        // The last of the list whose preceding mass is below target.
        if (g.me == 0) {
          const int per = (listed + kThreads - 1) / kThreads;
          uint64_t sum = 0, all;
          for (int e = 0; e < per; ++e) {
            const int i = tid * per + e;
            if (i < listed) sum += mass_of(weight(row, value_of((uint32_t)(s.list[i] >> 32))));
          }
          uint64_t before = above + cta_before(s, sum, all);
          for (int e = 0; e < per; ++e) {
            const int i = tid * per + e;
            if (i >= listed) break;
            const uint64_t m = mass_of(weight(row, value_of((uint32_t)(s.list[i] >> 32))));
            if (m && before < target && before + m >= target)
              for (int o = 0; o < g.n; ++o) g.of(o)->found[g.par][0] = s.list[i];
            before += m;
          }
        }
        g.sync();
        cut.key = (uint32_t)(s.found[g.par][0] >> 32);
        cut.last = (int)~(uint32_t)s.found[g.par][0];
        g.par ^= 1;
      } else if (exact) {
        uint32_t lo, hi;
        keys(bin, lo, hi);
        take(find_by_key<true>(g, x, row, within, max(lo, within.key), hi, above, target));
      } else {  // the estimate was off, or there were no bins
        take(find_by_key<true>(g, x, row, within, max(within.key, klow), kmax, 0, target));
      }
    }
  }

  // Running sums by index: (rank, level, warp, lane, element).
  // (min_p by the weight itself; below this by more than any rounding, not)
  const float cut_f = cut.key ? value_of(cut.key) : kNegInf;
  const float min_f = min_p > 0.f ? row.max + fminf(temp * (logf(min_p) - 0.01f), 0.f) - fabsf(row.max) * 1e-6f : kNegInf;
  const float least_kept = fmaxf(cut_f, min_f <= row.max ? min_f : kNegInf);
  const float floor_f = fmaxf(least_kept, row.low);
  auto candidate = [&](float f, int i) { return f >= floor_f && (f > cut_f || i <= cut.last); };
  auto kept_mass = [&](float f, int i) -> uint64_t {
    if (!candidate(f, i)) return 0;
    const double w = weight(row, f);
    return w >= (double)min_p || i == imax ? mass_of(w) : 0;
  };
  auto level_mass = [&](int l) -> uint64_t {
    float q[4];
    x.four(l, q);
    const int i = x.index(l);
    return kept_mass(q[0], i) + kept_mass(q[1], i + 1) + kept_mass(q[2], i + 2) + kept_mass(q[3], i + 3);
  };
  uint64_t sum = 0;
  __syncthreads();  // s.warp64 is free, s.table there
#pragma unroll 1
  for (int l = 0; l < a.levels; ++l) {
    const uint64_t m = level_mass(l);
    const uint64_t t = __any_sync(0xffffffffu, m != 0) ? warp_reduce(m, Add()) : 0;
    if (lane == 0) s_level[l * kWarps + warp] = t;
    sum += t;
  }
  if (lane == 0) s.warp64[warp] = sum;
  __syncthreads();
  if (tid < g.n) {
    uint64_t t = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += s.warp64[w];
    g.of(tid)->all_a[g.par][g.me] = t;
  }
  g.sync();
  uint64_t whole = 0, start = 0;
  for (int i = 0; i < g.n; ++i) {
    if (i < g.me) start += s.all_a[g.par][i];
    whole += s.all_a[g.par][i];
  }
  const uint64_t here = s.all_a[g.par][g.me];
  const uint64_t goal = goal_of(a.uniforms[r], whole);
  if (goal < start || goal >= start + here) return;
  uint64_t at = start;
  int l = 0;
  bool mine = false;
  for (; l < a.levels; ++l) {  // the level that passes the goal, then the warp
    uint64_t t = s_level[l * kWarps + (lane % kWarps)];
    uint64_t incl = warp_inclusive(lane < kWarps ? t : 0, lane);
    const uint64_t all = __shfl_sync(0xffffffffu, incl, kWarps - 1);
    if (goal < at + all) {
      const uint64_t before = at + __shfl_sync(0xffffffffu, incl - t, warp);
      const uint64_t own = __shfl_sync(0xffffffffu, t, warp);
      mine = goal >= before && goal < before + own;
      at = before;
      break;
    }
    at += all;
  }
  if (!mine) return;
  const uint64_t m = level_mass(l);
  at += warp_inclusive(m, lane) - m;
  if (goal < at || goal >= at + m) return;
  float f[4];
  x.four(l, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t t = kept_mass(f[e], x.index(l) + e);
    if (goal >= at && goal < at + t) a.ids[r] = x.index(l) + e;
    at += t;
  }
}

template <typename T, bool kKeep>
cudaError_t launch_rows(const SampleArgs& a, int64_t rows, int cluster, int smem, cudaStream_t stream) {
  const void* k = reinterpret_cast<const void*>(k_sample<T, kKeep>);
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
  // As many CTAs as run at once (two an SM), but a vector a thread at least;
  // more where the row would not stay in shared memory.
  const int64_t vectors = ((int64_t)p.vocab + 3) / 4;
  int cluster = 1;
  while (cluster < kMaxCluster && vectors > cluster * kThreads &&
         (p.rows * cluster * 2 <= 2 * device_sm_count() || vectors * 4 * elt > (int64_t)cluster * kKeepBytes))
    cluster *= 2;
  a.levels = (int)((vectors + (int64_t)cluster * kThreads - 1) / ((int64_t)cluster * kThreads));
  const int sums = (int)sizeof(Shared) + a.levels * kWarps * 8, part = a.levels * kThreads * 4 * elt;
  cudaError_t e;
  if (part <= kKeepBytes)
    e = elt == 2 ? launch_rows<uint16_t, true>(a, p.rows, cluster, sums + part, stream)
                 : launch_rows<float, true>(a, p.rows, cluster, sums + part, stream);
  else
    e = elt == 2 ? launch_rows<uint16_t, false>(a, p.rows, cluster, sums, stream)
                 : launch_rows<float, false>(a, p.rows, cluster, sums, stream);
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "sample_tokens launch");
}

}  // namespace wr
