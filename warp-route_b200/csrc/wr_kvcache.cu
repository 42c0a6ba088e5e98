// wr_kvcache.cu — keys and values of new tokens into a paged cache, with the
// position rotation applied on the way (and the queries rotated by the same
// angles).
//
//   a = position * inv_freq[i], i < rot_dim / 2
//   (x_i, x_j) -> (x_i cos a - x_j sin a, x_j cos a + x_i sin a)
//
// with j = i + rot_dim / 2, or pairs (2i, 2i + 1) when interleaved; the rest
// of the head passes through.  The angle is a 64-bit product reduced by whole
// turns in 64 bits (at position 1e6 a 32-bit product is off by 0.03 rad); the
// remainder's sine and cosine and the rotation are fp32, rounded once to the
// cache's type.
//
// The work is a copy, so HBM bounds it, and for one token latency.  One CTA
// takes one token (a slice of its heads when there are few tokens, so that a
// single token still spreads over the SMs); its sines and cosines are computed
// once into shared memory and serve every head.  A thread moves pairs of
// 16-byte chunks, the two of a pair half a rotation apart, so that each is
// read once; all its loads are on their way before the angles are computed
// and the slot is looked up.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "wr_common.cuh"
#include "wr_internal.h"

namespace wr {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendUnroll = 3;  // pairs of chunks a thread has in flight
constexpr int kMaxHeadDim = 256;

struct AppendArgs {
  const void *k, *v, *q;
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs;  // token and head strides, elements
  void *k_cache, *v_cache, *q_out;
  int64_t page_stride, head_stride, slot_stride;
  const int64_t* slots;
  const int64_t* positions;
  const float* inv_freq;
  int64_t num_slots;
  int hq, hkv, dim, rot, page_size, interleaved;
  int chunks;           // 16-byte chunks a head
  int apart;            // chunks between the two of a pair that turns (half a rotation); 0: neighbours
  int pairs, pairs_v;   // pairs of a head of q or k, and of v
  uint32_t pairs_inv, pairs_v_inv;  // ceil(2^32 / pairs), for the division; 0: one pair
  int pairs_per_cta;    // of one token
};

WR_DEVINL float ld_elem(const uint16_t* p) { return bf16lo(*p); }
WR_DEVINL float ld_elem(const float* p) { return *p; }

WR_DEVINL uint4 pack_chunk(const float (&f)[8], const uint16_t*) {
  uint4 r;
  uint32_t* w = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&b);
  }
  return r;
}
WR_DEVINL uint4 pack_chunk(const float (&f)[4], const float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}

// kApart: half a rotation is a whole number of chunks; a pair then holds both
// partners of its columns.  Otherwise pairs are neighbours, and for halves
// that end inside a chunk the partner columns are read one by one.
template <typename T, bool kApart>
__global__ void __launch_bounds__(kAppendThreads) k_append_paged_kv(AppendArgs a) {
  constexpr int V = Chunk<T>::kVec;
  __shared__ float s_cos[kMaxHeadDim / 2], s_sin[kMaxHeadDim / 2];
  __shared__ int64_t s_row;  // element offset of this token's cache row, -1: none
  const int64_t t = blockIdx.x;
  const int half = a.rot >> 1;
  const int nq = a.hq * a.pairs, nk = a.hkv * a.pairs;
  const int total = nq + nk + a.hkv * a.pairs_v;
  const int first = blockIdx.y * a.pairs_per_cta;
  const int last = min(total, first + a.pairs_per_cta);
  bool ready = false;
  for (int i0 = first + threadIdx.x; i0 < last || !ready; i0 += kAppendThreads * kAppendUnroll) {
    uint4 x0[kAppendUnroll], x1[kAppendUnroll];
    int head[kAppendUnroll], c0[kAppendUnroll], c1[kAppendUnroll];  // c1 < 0: no second chunk
    int part[kAppendUnroll];  // 0: q, 1: k, 2: v, -1: nothing
    const T* src[kAppendUnroll];
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      int i = i0 + u * kAppendThreads;
      part[u] = i >= last ? -1 : (i < nq ? 0 : (i < nq + nk ? 1 : 2));
      if (part[u] < 0) continue;
      i -= part[u] == 0 ? 0 : (part[u] == 1 ? nq : nq + nk);
      const bool v = part[u] == 2;
      const uint32_t inv = v ? a.pairs_v_inv : a.pairs_inv;
      const int h = inv ? (int)__umulhi((uint32_t)i, inv) : i;
      const int j = i - h * (v ? a.pairs_v : a.pairs);
      head[u] = h;
      if (kApart && !v && j < a.apart) {
        c0[u] = j;
        c1[u] = j + a.apart;
      } else {  // neighbours, behind the columns that turn
        c0[u] = (kApart && !v ? 2 * a.apart + 2 * (j - a.apart) : 2 * j);
        c1[u] = c0[u] + 1 < a.chunks ? c0[u] + 1 : -1;
      }
      const void* base = part[u] == 0 ? a.q : (part[u] == 1 ? a.k : a.v);
      const int64_t ts = part[u] == 0 ? a.q_ts : (part[u] == 1 ? a.k_ts : a.v_ts);
      const int64_t hs = part[u] == 0 ? a.q_hs : (part[u] == 1 ? a.k_hs : a.v_hs);
      src[u] = static_cast<const T*>(base) + t * ts + h * hs;
      x0[u] = ldg_nc_v4(src[u] + c0[u] * V);
      if (c1[u] >= 0) x1[u] = ldg_nc_v4(src[u] + c1[u] * V);
    }
    if (!ready) {
      ready = true;
      if (threadIdx.x == kAppendThreads - 1) {
        const int64_t slot = a.slots[t];
        int64_t row = -1;
        if (slot >= 0 && slot < a.num_slots) {
          const int64_t page = (uint64_t)slot >> 32 ? slot / a.page_size
                                                    : (int64_t)((uint32_t)slot / (uint32_t)a.page_size);
          row = page * a.page_stride + (slot - page * a.page_size) * a.slot_stride;
        }
        s_row = row;
      }
      for (int i = threadIdx.x; i < half; i += kAppendThreads) {
        double turns = (double)a.positions[t] * (double)a.inv_freq[i] * 0.15915494309189533577;
        turns -= rint(turns);
        sincospif(2.0f * (float)turns, &s_sin[i], &s_cos[i]);
      }
      __syncthreads();
    }
    const int64_t row = s_row;
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      if (part[u] < 0 || (part[u] > 0 && row < 0)) continue;
      if (part[u] < 2 && c0[u] * V < a.rot) {
        float x[V], y[V];
        Chunk<T>::widen(x0[u], x);
        if (c1[u] >= 0) Chunk<T>::widen(x1[u], y);
        if (kApart) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float cs = s_cos[c0[u] * V + e], sn = s_sin[c0[u] * V + e];
            const float p = x[e], r = y[e];
            x[e] = p * cs - r * sn;
            y[e] = r * cs + p * sn;
          }
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (w == 1 && c1[u] < 0) continue;
            float* f = w ? y : x;
            const int c = (w ? c1[u] : c0[u]) * V;
            if (a.interleaved) {
#pragma unroll
              for (int e = 0; e < V; e += 2)
                if (c + e < a.rot) {
                  const float cs = s_cos[(c + e) >> 1], sn = s_sin[(c + e) >> 1];
                  const float p = f[e], r = f[e + 1];
                  f[e] = p * cs - r * sn;
                  f[e + 1] = r * cs + p * sn;
                }
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e)
                if (c + e < a.rot) {
                  const bool lo = c + e < half;
                  const int k = lo ? c + e : c + e - half;
                  const float p = ld_elem(src[u] + (lo ? c + e + half : c + e - half));
                  f[e] = f[e] * s_cos[k] + (lo ? -p : p) * s_sin[k];
                }
            }
          }
        }
        x0[u] = pack_chunk(x, src[u]);
        if (c1[u] >= 0) x1[u] = pack_chunk(y, src[u]);
      }
      T* out = part[u] == 0 ? static_cast<T*>(a.q_out) + (t * a.hq + head[u]) * a.dim
                            : static_cast<T*>(part[u] == 1 ? a.k_cache : a.v_cache) + row + head[u] * a.head_stride;
      *reinterpret_cast<uint4*>(out + c0[u] * V) = x0[u];
      if (c1[u] >= 0) *reinterpret_cast<uint4*>(out + c1[u] * V) = x1[u];
    }
  }
}

}  // namespace

wr_status_t launch_append(const AppendProblem& p, cudaStream_t stream) {
  AppendArgs a{};
  a.k = p.k; a.v = p.v; a.q = p.q;
  a.k_ts = p.k_ts; a.k_hs = p.k_hs; a.v_ts = p.v_ts; a.v_hs = p.v_hs; a.q_ts = p.q_ts; a.q_hs = p.q_hs;
  a.k_cache = p.c.k; a.v_cache = p.c.v; a.q_out = p.q_out;
  a.page_stride = p.c.page_stride; a.head_stride = p.c.head_stride; a.slot_stride = p.c.slot_stride;
  a.slots = p.slots; a.positions = p.positions; a.inv_freq = p.inv_freq;
  a.num_slots = (int64_t)p.c.num_pages * p.c.page_size;
  a.hq = p.hq; a.hkv = p.c.hkv; a.dim = p.c.dim; a.rot = p.rot; a.page_size = p.c.page_size;
  a.interleaved = p.interleaved;
  const int elt = p.c.dtype == WR_DTYPE_BF16 ? 2 : 4;
  a.chunks = p.c.dim * elt / 16;
  const int half_bytes = (p.rot / 2) * elt;
  const bool apart = !p.interleaved && p.rot > 0 && half_bytes % 16 == 0;
  a.apart = apart ? half_bytes / 16 : 0;
  a.pairs = a.apart + (a.chunks - 2 * a.apart + 1) / 2;
  a.pairs_v = (a.chunks + 1) / 2;
  auto inverse = [](int n) { return n == 1 ? 0u : (uint32_t)(((1ull << 32) + n - 1) / n); };
  a.pairs_inv = inverse(a.pairs);
  a.pairs_v_inv = inverse(a.pairs_v);
  const int total = p.hq * a.pairs + p.c.hkv * (a.pairs + a.pairs_v);
  // Few tokens: a CTA takes one pair a thread, so that the token spreads over
  // several SMs; many tokens: whole tokens, whose sines are then computed once.
  const int slices = (int64_t)p.T * 4 <= device_sm_count() ? (total + kAppendThreads - 1) / kAppendThreads : 1;
  a.pairs_per_cta = (total + slices - 1) / slices;
  const dim3 grid((unsigned)p.T, (unsigned)slices);
  if (elt == 2) {
    if (apart) k_append_paged_kv<uint16_t, true><<<grid, kAppendThreads, 0, stream>>>(a);
    else k_append_paged_kv<uint16_t, false><<<grid, kAppendThreads, 0, stream>>>(a);
  } else {
    if (apart) k_append_paged_kv<float, true><<<grid, kAppendThreads, 0, stream>>>(a);
    else k_append_paged_kv<float, false><<<grid, kAppendThreads, 0, stream>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "append_paged_kv launch");
}

}  // namespace wr
