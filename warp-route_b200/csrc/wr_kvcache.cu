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
// The work is a copy, so HBM bounds it.  One CTA takes one token (a slice of
// its heads when there are few tokens, so that a single token still spreads
// over the SMs); its sines and cosines are computed once into shared memory
// and serve every head.  A thread moves 16-byte chunks, several in flight:
// the chunk and, for the rotation, its partner half a rotation away, which
// another thread of the CTA reads too (the second read hits L1).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "wr_common.cuh"
#include "wr_internal.h"

namespace wr {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendUnroll = 4;  // chunks a thread has in flight
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
  int chunks;           // 16-byte chunks per head
  uint32_t chunks_inv;  // ceil(2^32 / chunks)
  int chunks_per_cta;   // chunks of one token that one CTA moves
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

// kPairVec: half a rotation is a whole number of chunks, so a chunk's
// partners are one chunk too (read with one load; else element by element).
template <typename T, bool kPairVec>
__global__ void __launch_bounds__(kAppendThreads) k_append_paged_kv(AppendArgs a) {
  constexpr int V = Chunk<T>::kVec;
  __shared__ float s_cos[kMaxHeadDim / 2], s_sin[kMaxHeadDim / 2];
  __shared__ int64_t s_row;  // element offset of this token's cache row, -1: none
  const int64_t t = blockIdx.x;
  const int half = a.rot >> 1;
  if (threadIdx.x == kAppendThreads - 1) {
    const int64_t slot = a.slots[t];
    int64_t row = -1;
    if (slot >= 0 && slot < a.num_slots) {
      const int64_t page = slot / a.page_size;
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
  const int64_t row = s_row;
  const int nq = a.hq * a.chunks, nk = a.hkv * a.chunks;
  const int total = nq + 2 * nk;
  const int first = blockIdx.y * a.chunks_per_cta;
  const int last = min(total, first + a.chunks_per_cta);
  for (int i0 = first + threadIdx.x; i0 < last; i0 += kAppendThreads * kAppendUnroll) {
    uint4 own[kAppendUnroll], other[kAppendUnroll];
    const T* src[kAppendUnroll];
    T* dst[kAppendUnroll];
    int col[kAppendUnroll];  // first column of the chunk; -1: nothing to do
    bool turn[kAppendUnroll];
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      int i = i0 + u * kAppendThreads;
      col[u] = -1;
      turn[u] = false;
      if (i >= last) continue;
      const T* base;
      int64_t hs;
      T* out;
      int64_t ohs;
      bool rotates = true;
      if (i < nq) {
        base = static_cast<const T*>(a.q) + t * a.q_ts;
        hs = a.q_hs;
        out = static_cast<T*>(a.q_out) + t * (int64_t)a.hq * a.dim;
        ohs = a.dim;
      } else {
        if (row < 0) continue;
        i -= nq;
        rotates = i < nk;
        if (rotates) {
          base = static_cast<const T*>(a.k) + t * a.k_ts;
          hs = a.k_hs;
          out = static_cast<T*>(a.k_cache) + row;
        } else {
          i -= nk;
          base = static_cast<const T*>(a.v) + t * a.v_ts;
          hs = a.v_hs;
          out = static_cast<T*>(a.v_cache) + row;
        }
        ohs = a.head_stride;
      }
      const int h = __umulhi((uint32_t)i, a.chunks_inv);
      const int c = (i - h * a.chunks) * V;
      col[u] = c;
      turn[u] = rotates && c < a.rot;
      src[u] = base + h * hs;
      dst[u] = out + h * ohs + c;
      own[u] = ldg_nc_v4(src[u] + c);
      if (kPairVec && turn[u] && !a.interleaved)
        other[u] = *reinterpret_cast<const uint4*>(src[u] + (c < half ? c + half : c - half));
    }
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      if (col[u] < 0) continue;
      if (turn[u]) {
        float x[V], y[V];
        Chunk<T>::widen(own[u], x);
        const int c = col[u];
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            if (c + e < a.rot) {
              const float cs = s_cos[(c + e) >> 1], sn = s_sin[(c + e) >> 1];
              const float p = x[e], r = x[e + 1];
              x[e] = p * cs - r * sn;
              x[e + 1] = r * cs + p * sn;
            }
          }
        } else {
          if (kPairVec) Chunk<T>::widen(other[u], y);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int j = c + e;
            if (j < a.rot) {
              const bool lo = j < half;
              const int p = lo ? j : j - half;
              const float yy = kPairVec ? y[e] : ld_elem(src[u] + (lo ? j + half : j - half));
              x[e] = x[e] * s_cos[p] + (lo ? -yy : yy) * s_sin[p];
            }
          }
        }
        own[u] = pack_chunk(x, src[u]);
      }
      *reinterpret_cast<uint4*>(dst[u]) = own[u];
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
  a.chunks_inv = (uint32_t)(((1ull << 32) + a.chunks - 1) / a.chunks);
  if (a.chunks == 1) a.chunks_inv = 0xffffffffu;
  const int total = (p.hq + 2 * p.c.hkv) * a.chunks;
  // Few tokens: a CTA takes one chunk a thread, so that the token spreads
  // over several SMs and no thread loops; many tokens: whole tokens, whose
  // sines are then computed once.
  const int slices = (int64_t)p.T * 4 <= device_sm_count() ? (total + kAppendThreads - 1) / kAppendThreads : 1;
  a.chunks_per_cta = (total + slices - 1) / slices;
  const dim3 grid((unsigned)p.T, (unsigned)slices);
  const bool vec = (a.rot / 2) * elt % 16 == 0 || a.interleaved;
  if (elt == 2) {
    if (vec) k_append_paged_kv<uint16_t, true><<<grid, kAppendThreads, 0, stream>>>(a);
    else k_append_paged_kv<uint16_t, false><<<grid, kAppendThreads, 0, stream>>>(a);
  } else {
    if (vec) k_append_paged_kv<float, true><<<grid, kAppendThreads, 0, stream>>>(a);
    else k_append_paged_kv<float, false><<<grid, kAppendThreads, 0, stream>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "append_paged_kv launch");
}

}  // namespace wr
