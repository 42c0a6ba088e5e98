// wr_attention.cu — attention of a batch over a paged cache, with a prefix
// shared by all sequences.
//
//   s_j = scale * q . k_j over the prefix and the sequence's own keys up to
//         the token's own;   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
//
// by the running maximum m and sum l, in units of log2 (2^(s log2(e) - m));
// scores, m, l and the sums O are fp32, the weights 2^(s - m) are rounded to
// the cache's type for the second product (bf16: half a step of 2^-8, as the
// output itself), l adds them before that rounding.
//
// Own keys: each sequence's few rows meet its own keys, one byte of cache for
// a few operations, so HBM bounds it.  k_attn_stream: a warp works alone on
// 16 keys at a time, which it brings with 16-byte asynchronous copies into
// a ring of its own in shared memory (no barrier between warps anywhere), and
// multiplies with its 16 rows by mma.sync (the M of tcgen05 is 128 rows, of
// which these segments fill 1 to 16; nothing here comes near the tensor
// rate).  The units of all sequences are dealt to the warps evenly (see
// wr_attention.cuh), so one long sequence and hundreds of short ones fill the
// GPU alike.  k_attn_stream_f32: the same ring and split with fp32 products
// on the CUDA cores, 4 or 8 rows a warp.
//
// Prefix: its rows are the tokens of all sequences.  With one sequence, or a
// prefix short enough, each sequence reads it with its own keys; else it is a
// segment of its own, whose partial results k_attn_combine joins to those of
// the own keys: m = max m_s, l = sum l_s 2^(m_s - m), O = sum O_s 2^(m_s - m),
// in the order of the pieces, so that a call's result is the same each time.
#include <climits>

#include "wr_attention.cuh"

namespace wr {
namespace {

// A CTA is one warp: no warp needs another, and the hardware fills an SM with
// as many as it has room for.  (Beside a CTA of the prefix's kernel a warp of
// this one gained nothing: its mma.sync wait for the tensor core, 184 us for
// keys that take 60 alone.)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
#define WR_NEG_INF (-__int_as_float(0x7f800000))

WR_DEVINL float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
WR_DEVINL void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
WR_DEVINL void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
WR_DEVINL void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

WR_DEVINL void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
WR_DEVINL void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
WR_DEVINL void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
WR_DEVINL uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}

// ---------------------------------------------------------------------------
// The split, computed by each warp from the lengths
// ---------------------------------------------------------------------------
template <int MR>
WR_DEVINL int64_t seg_units(const AttnArgs& a, int i) {
  if (i >= segments(a)) return 0;
  const Segment s = segment(a, i);
  return (int64_t)a.hkv * row_tiles<MR>(a, s) * key_units(s);
}

// Units of the launch: a warp adds them up, 32 segments at a time.
template <int MR>
WR_DEVINL int64_t all_units(const AttnArgs& a, int lane) {
  int64_t sum = 0;
#pragma unroll 4
  for (int i = lane; i < segments(a); i += 32) sum += seg_units<MR>(a, i);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return sum;
}

WR_DEVINL int64_t warp_before(int64_t v, int lane, int64_t& all) {
  int64_t incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += u;
  }
  all = __shfl_sync(0xffffffffu, incl, 31);
  return incl - v;
}

// The sequence that token t belongs to, -1: none.
WR_DEVINL int seq_of(const AttnArgs& a, int t) {
  int lo = 0, hi = a.B;  // last b with q_start[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.q_start + mid) <= t) lo = mid; else hi = mid;
  }
  const Segment s = segment(a, lo + (a.lead > 0));
  return t >= s.q0 && t < s.q0 + s.nq ? lo : -1;
}

// What the joining kernel reads: the first unit of each segment, by warp 0,
// and the sequence of each token, by all.
template <int MR>
WR_DEVINL void write_index(const AttnArgs& a, int lane) {
  if (blockIdx.x == 0) {
    int64_t base = 0, all;
    for (int i0 = 0; i0 < segments(a); i0 += 32) {
      const int64_t at = base + warp_before(seg_units<MR>(a, i0 + lane), lane, all);
      if (i0 + lane < segments(a)) a.seg_unit[i0 + lane] = at;
      base += all;
    }
    if (lane == 0) a.seg_unit[segments(a)] = base;
  }
  if (a.q_start)
    for (int t = blockIdx.x * 32 + lane; t < a.T; t += gridDim.x * 32) a.token_seq[t] = seq_of(a, t);
}

// A position in the order of the units.
template <int MR>
struct Cursor {
  int b, h, rt, u;   // segment, key head, row tile, unit
  int rts, us;       // row tiles and units of the segment
  Segment s;

  WR_DEVINL void load(const AttnArgs& a) {
    s = segment(a, b);
    rts = row_tiles<MR>(a, s);
    us = key_units(s);
  }
  // To unit `at` (< units of the launch).
  WR_DEVINL void seek(const AttnArgs& a, int lane, int64_t at) {
    for (int i0 = 0;; i0 += 32) {
      int64_t all;
      const int64_t v = seg_units<MR>(a, i0 + lane), before = warp_before(v, lane, all);
      const uint32_t past = __ballot_sync(0xffffffffu, before + v > at);
      if (past) {
        const int first = __ffs(past) - 1;
        b = i0 + first;
        at -= __shfl_sync(0xffffffffu, before, first);
        break;
      }
      at -= all;
    }
    load(a);
    const int64_t tile = quotient(at, us);
    u = (int)(at - tile * us);
    h = (int)quotient(tile, rts);
    rt = (int)(tile - (int64_t)h * rts);
  }
  // Never called past the launch's last unit.
  WR_DEVINL void next(const AttnArgs& a) {
    if (++u < us) return;
    u = 0;
    if (++rt < rts) return;
    rt = 0;
    if (++h < a.hkv) return;
    h = 0;
    do {
      ++b;
      load(a);
    } while (rts == 0 && b + 1 < segments(a));
  }
};

// The page of this lane's key of a unit, read ahead of the copies.
template <int MR>
WR_DEVINL int lane_page(const AttnArgs& a, const Cursor<MR>& c, int lane) {
  const int j = c.u * kUnitTokens + (lane & 15);
  int page, row;
  if (j < c.s.prefix) {
    split_page(j, a.page_size, a.page_shift, page, row);
    return __ldg(a.prefix_pages + page);
  }
  const int jj = j - c.s.prefix;
  if (jj >= c.s.len) return -1;
  split_page(jj, a.page_size, a.page_shift, page, row);
  return __ldg(a.tables + (c.b - (a.lead > 0)) * a.table_stride + page);
}

// Offset (elements) of this lane's key in the cache; its valid bit.  A page
// outside the cache makes its keys invisible.
template <int MR>
WR_DEVINL int64_t lane_offset(const AttnArgs& a, const Cursor<MR>& c, int page, int lane, bool& ok) {
  const int j = c.u * kUnitTokens + (lane & 15);
  int p, row;
  split_page(j < c.s.prefix ? j : j - c.s.prefix, a.page_size, a.page_shift, p, row);
  ok = page >= 0 && page < a.num_pages;
  return ok ? page * a.page_stride + c.h * a.head_stride + row * a.slot_stride : 0;
}

// Number of keys that row (token i of the sequence) sees of the segment.
template <int MR>
WR_DEVINL int row_limit(const AttnArgs& a, const Cursor<MR>& c, int i) {
  return c.s.prefix + max(0, c.s.len - c.s.nq + i + 1);
}

// The first unit with a key that some row of the tile does not see, because a
// later token of its sequence put it there.  A weight of zero does not hide an
// infinity or a NaN in that key's value: from here on the values are looked
// through, and a unit that holds one is added up key by key, by the rows that
// see the key.
template <int MR>
WR_DEVINL int first_cut(const AttnArgs& a, const Cursor<MR>& c) {
  if (c.s.nq <= 1) return INT_MAX;
  return (c.s.prefix + max(0, c.s.len - c.s.nq + c.rt * MR / a.group + 1)) / kUnitTokens;
}

// ---------------------------------------------------------------------------
// bf16
// ---------------------------------------------------------------------------
constexpr int kStages = 3;
template <int DP>
struct StreamCfg {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kTile = kUnitTokens * kRowBytes;  // K (or V) of a unit
  static constexpr bool kQSmem = DP > 128;  // the fragments of 256 columns do not fit beside O
  static constexpr int kSmem = kStages * 2 * kTile + (kQSmem ? kTile : 0);
};

// Registers for as many warps an SM as the rings leave room for.
// kSeveral: some sequence may have several tokens.  The look at their later
// values costs such calls 2 to 14 % (24 sequences of 1 to 9: 67.8 us, 66.1
// without; the 209 sequences of 1 to 64 below: 257, 226).
template <int DP, bool kSeveral>
__global__ void __launch_bounds__(32) __maxnreg__(DP == 64 ? 128 : DP == 128 ? 224 : 255) k_attn_stream(const AttnArgs a) {
  using C = StreamCfg<DP>;
  constexpr int MR = 16, CPR = DP / 8, RPP = 32 / CPR;  // chunks a row, rows a pass of the warp
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint32_t s_bits[kStages];
  const int lane = threadIdx.x;
  griddep_launch_dependents();
  AttnSplit sp;
  sp.units = all_units<MR>(a, lane);
  sp.ranges = min((int64_t)gridDim.x, sp.units);
  const int64_t w = blockIdx.x;
  if (w < sp.ranges) {
    const int64_t u0 = range_start(sp, w), u1 = range_start(sp, w + 1);
    const uint32_t ring_s = smem_u32(ring);
    const uint32_t q_s = ring_s + kStages * 2 * C::kTile;
    Cursor<MR> cl, cc;  // the copies' and the products' position
    cl.seek(a, lane, u0);
    cc = cl;
    const int n = (int)(u1 - u0);
    int page = lane_page(a, cl, lane);
    int loaded = 0;
    auto load = [&]() {
      if (loaded < n) {
        const int st = loaded % kStages;
        bool ok;
        const int64_t off = lane_offset(a, cl, page, lane, ok);
        const uint32_t bits = __ballot_sync(0xffffffffu, ok) & 0xffffu;
        if (lane == 0) s_bits[st] = bits;
        const uint32_t base = ring_s + st * 2 * C::kTile;
        const int c = lane % CPR;
        const bool in = c * 8 < a.dim;
#pragma unroll
        for (int i = 0; i < kUnitTokens / RPP; ++i) {
          const int r = i * RPP + lane / CPR;
          const int64_t o = __shfl_sync(0xffffffffu, off, r) + (in ? c * 8 : 0);
          const uint32_t bytes = in && ((bits >> r) & 1) ? 16 : 0;  // 0: the chunk is filled with zeros
          const uint32_t d = base + r * C::kRowBytes + ((c ^ (r & 7)) << 4);
          cp_async16(d, static_cast<const uint16_t*>(a.kc) + o, bytes);
          cp_async16(d + C::kTile, static_cast<const uint16_t*>(a.vc) + o, bytes);
        }
        ++loaded;
        if (loaded < n) {
          cl.next(a);
          page = lane_page(a, cl, lane);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load();
    write_index<MR>(a, lane);

    uint32_t qf[C::kQSmem ? 1 : DP / 16][4];
    float o[DP / 8][4];
    float m0 = WR_NEG_INF, m1 = WR_NEG_INF, l0 = 0.f, l1 = 0.f;
    int lim0 = 0, lim1 = 0, first = 0, cut = 0;
    const int g8 = lane >> 2, c2 = (lane & 3) * 2;
    for (int it = 0; it < n; ++it) {
      __syncwarp();  // every lane has read what the next copies overwrite
      load();
      if (it == 0 || cc.u == 0) {  // a new piece
        first = cc.u;
        if constexpr (kSeveral) cut = first_cut(a, cc);
        m0 = m1 = WR_NEG_INF;
        l0 = l1 = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
        const int r0 = cc.rt * MR + g8, r1 = r0 + 8, rows = cc.s.nq * a.group;
        const int i0 = r0 / a.group, i1 = r1 / a.group;
        lim0 = row_limit(a, cc, i0);
        lim1 = row_limit(a, cc, i1);
        const uint16_t* qb = static_cast<const uint16_t*>(a.q);
        const uint16_t* q0 = qb + (int64_t)(cc.s.q0 + i0) * a.q_ts +
                             (int64_t)(cc.h * a.group + r0 - i0 * a.group) * a.q_hs;
        const uint16_t* q1 = qb + (int64_t)(cc.s.q0 + i1) * a.q_ts +
                             (int64_t)(cc.h * a.group + r1 - i1 * a.group) * a.q_hs;
        if constexpr (C::kQSmem) {
          for (int i = lane; i < MR * CPR; i += 32) {
            const int r = i / CPR, c = i % CPR, rr = cc.rt * MR + r, ii = rr / a.group;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (rr < rows && c * 8 < a.dim)
              v = *reinterpret_cast<const uint4*>(qb + (int64_t)(cc.s.q0 + ii) * a.q_ts +
                                                  (int64_t)(cc.h * a.group + rr - ii * a.group) * a.q_hs +
                                                  c * 8);
            *reinterpret_cast<uint4*>(ring + kStages * 2 * C::kTile + r * C::kRowBytes +
                                      ((c ^ (r & 7)) << 4)) = v;
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const int d0 = k * 16 + c2, d1 = d0 + 8;
            auto at = [&](const uint16_t* p, int r, int d) {
              return r < rows && d < a.dim ? *reinterpret_cast<const uint32_t*>(p + d) : 0u;
            };
            qf[k][0] = at(q0, r0, d0);
            qf[k][1] = at(q1, r1, d0);
            qf[k][2] = at(q0, r0, d1);
            qf[k][3] = at(q1, r1, d1);
          }
        }
      }
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const int st = it % kStages;
      const uint32_t kb = ring_s + st * 2 * C::kTile, vb = kb + C::kTile;
      const uint32_t bits = s_bits[st];
      float s[2][4] = {};
      {
        const int r = ((lane >> 4) << 3) + (lane & 7);
        const uint32_t row = kb + r * C::kRowBytes;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t f[4];
          ldsm4(f, row + (((2 * k + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
          if constexpr (C::kQSmem) {
            uint32_t qq[4];
            const int qr = lane & 15;
            ldsm4(qq, q_s + qr * C::kRowBytes + (((2 * k + (lane >> 4)) ^ (qr & 7)) << 4));
            mma16816(s[0], qq, f[0], f[1]);
            mma16816(s[1], qq, f[2], f[3]);
          } else {
            mma16816(s[0], qf[k], f[0], f[1]);
            mma16816(s[1], qf[k], f[2], f[3]);
          }
        }
      }
      const int j0 = cc.u * kUnitTokens;
      float mx0 = WR_NEG_INF, mx1 = WR_NEG_INF;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = h * 8 + c2 + e;
          const bool vis = (bits >> j) & 1;
          s[h][e] = vis && j0 + j < lim0 ? s[h][e] * a.scale_log2 : WR_NEG_INF;
          s[h][2 + e] = vis && j0 + j < lim1 ? s[h][2 + e] * a.scale_log2 : WR_NEG_INF;
          mx0 = fmaxf(mx0, s[h][e]);
          mx1 = fmaxf(mx1, s[h][2 + e]);
        }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
      }
      if (__any_sync(0xffffffffu, mx0 > m0 || mx1 > m1)) {
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        const float f0 = m0 == n0 ? 1.f : ex2(m0 - n0), f1 = m1 == n1 ? 1.f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[d][0] *= f0; o[d][1] *= f0;
          o[d][2] *= f1; o[d][3] *= f1;
        }
      }
      const float b0 = m0 == WR_NEG_INF ? 0.f : m0, b1 = m1 == WR_NEG_INF ? 0.f : m1;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[h][e] = ex2(s[h][e] - b0);
          s[h][2 + e] = ex2(s[h][2 + e] - b1);
          l0 += s[h][e];
          l1 += s[h][2 + e];
        }
      const uint32_t p[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]),
                             pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
      bool odd = false;
      if (kSeveral && cc.u >= cut) {
        uint32_t x = 0;  // an exponent of ones plus one carries into the sign
        auto look = [&](uint32_t v) { x |= (v & 0x7f807f80u) + 0x00800080u; };
#pragma unroll 4
        for (int i = lane; i < C::kTile / 16; i += 32) {
          const uint4 v = *reinterpret_cast<const uint4*>(ring + (st * 2 + 1) * C::kTile + i * 16);
          look(v.x); look(v.y); look(v.z); look(v.w);
        }
        odd = __any_sync(0xffffffffu, x & 0x80008000u);
      }
      if (odd) {
#pragma unroll 1
        for (int j = 0; j < kUnitTokens; ++j) {
          const int src = (lane & ~3) | ((j & 7) >> 1);
          const float p0 = __shfl_sync(0xffffffffu, j & 8 ? (j & 1 ? s[1][1] : s[1][0]) : (j & 1 ? s[0][1] : s[0][0]), src);
          const float p1 = __shfl_sync(0xffffffffu, j & 8 ? (j & 1 ? s[1][3] : s[1][2]) : (j & 1 ? s[0][3] : s[0][2]), src);
          const uint8_t* vr = ring + (st * 2 + 1) * C::kTile + j * C::kRowBytes + c2 * 2;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(vr + ((d ^ (j & 7)) << 4));
            const float lo = __uint_as_float(x << 16), hi = __uint_as_float(x & 0xffff0000u);
            if (j0 + j < lim0) {
              o[d][0] += p0 * lo;
              o[d][1] += p0 * hi;
            }
            if (j0 + j < lim1) {
              o[d][2] += p1 * lo;
              o[d][3] += p1 * hi;
            }
          }
        }
      } else {
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7);
        const uint32_t row = vb + r * C::kRowBytes;
#pragma unroll
        for (int c = 0; c < CPR; c += 2) {
          uint32_t f[4];
          ldsm4_t(f, row + (((c + (lane >> 4)) ^ (r & 7)) << 4));
          mma16816(o[c], p, f[0], f[1]);
          mma16816(o[c + 1], p, f[2], f[3]);
        }
      }
      const bool tile_end = cc.u == cc.us - 1;
      if (tile_end || it == n - 1) {  // the piece ends
        float t0 = l0, t1 = l1;
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          t0 += __shfl_xor_sync(0xffffffffu, t0, d);
          t1 += __shfl_xor_sync(0xffffffffu, t1, d);
        }
        const bool whole = tile_end && first == 0, lead = a.lead > 0 && cc.b == 0;
        const int rows = cc.s.nq * a.group;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int rl = g8 + half * 8, r = cc.rt * MR + rl;
          if (r >= rows) continue;
          const float mm = half ? m1 : m0, ll = half ? t1 : t0;
          const int i = r / a.group;
          const int64_t orow = (int64_t)(cc.s.q0 + i) * a.hq + cc.h * a.group + (r - i * a.group);
          if (whole && a.direct) {
            const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);  // NaN stays
            uint16_t* op = static_cast<uint16_t*>(a.out) + orow * a.dim;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d)
              if (d * 8 + c2 < a.dim)
                *reinterpret_cast<uint32_t*>(op + d * 8 + c2) =
                    pack_bf16(o[d][2 * half] * inv, o[d][2 * half + 1] * inv);
            if (a.lse && (lane & 3) == 0) a.lse[orow] = ll == 0.f ? WR_NEG_INF : (mm + log2f(ll)) * kLn2;
          } else {
            const int64_t prow = (w * 2 + (first == 0 ? 1 : 0)) * MR + rl;
            float* op = !whole ? a.part.piece + prow * a.dim : (lead ? a.lead_home : a.home) + orow * a.dim;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d)
              if (d * 8 + c2 < a.dim)
                *reinterpret_cast<float2*>(op + d * 8 + c2) = make_float2(o[d][2 * half], o[d][2 * half + 1]);
            if ((lane & 3) == 0)
              *(!whole ? a.part.piece_ml + prow : (lead ? a.lead_home_ml : a.home_ml) + orow) = make_float2(mm, ll);
          }
        }
      }
      if (it + 1 < n) cc.next(a);
    }
    cp_async_wait<0>();
    if (kSeveral && a.ends && lane == 0)
      a.ends[w] = make_int4(cc.b, cc.h, cc.rt, cc.u == cc.us - 1 || first > 0 ? -1 : cc.u);
  } else {
    write_index<MR>(a, lane);
  }
  griddep_wait();  // this launch counts as complete only after the one before it
}

// ---------------------------------------------------------------------------
// fp32
// ---------------------------------------------------------------------------
// Two stages: six warps an SM rather than four count for more than a third
// stage (12 sequences, 16 heads: 39 us against 43).
template <int DP, int MR>
struct StreamF32Cfg {
  static constexpr int kStages = 2;
  static constexpr int kMR = MR;
  static constexpr int kRowBytes = DP * 4;
  static constexpr int kTile = kUnitTokens * kRowBytes;
  static constexpr int kQBytes = kMR * kRowBytes;
  static constexpr int kPBytes = kUnitTokens * kMR * 4;
  static constexpr int kSmem = kStages * 2 * kTile + kQBytes + kPBytes;
};

// Lane (t, half) of the first product: key t of the unit, half the columns;
// of the second: DP / 32 columns, all keys.  K chunks are swizzled by key, so
// that the 8 lanes of a 16-byte read phase meet 8 different banks; Q and the
// weights are read by all lanes at once.
template <int DP, int MR, bool kSeveral>
__global__ void __launch_bounds__(32) k_attn_stream_f32(const AttnArgs a) {
  using C = StreamF32Cfg<DP, MR>;
  constexpr int kStages = C::kStages, CPR = DP / 4, HR = MR / 2;  // rows whose statistics a half of the lanes keeps
  constexpr int VC = DP / 32;  // columns of O a lane has
  constexpr int VW = VC < 4 ? VC : 4;  // ... in runs of VW
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint32_t s_bits[kStages];
  const int lane = threadIdx.x;
  griddep_launch_dependents();
  AttnSplit sp;
  sp.units = all_units<MR>(a, lane);
  sp.ranges = min((int64_t)gridDim.x, sp.units);
  const int64_t w = blockIdx.x;
  if (w < sp.ranges) {
    const int64_t u0 = range_start(sp, w), u1 = range_start(sp, w + 1);
    const uint32_t ring_s = smem_u32(ring);
    float* qs = reinterpret_cast<float*>(ring + kStages * 2 * C::kTile);
    float* ps = qs + MR * DP;
    Cursor<MR> cl, cc;
    cl.seek(a, lane, u0);
    cc = cl;
    const int n = (int)(u1 - u0);
    int page = lane_page(a, cl, lane);
    int loaded = 0;
    auto load = [&]() {
      if (loaded < n) {
        const int st = loaded % kStages;
        bool ok;
        const int64_t off = lane_offset(a, cl, page, lane, ok);
        const uint32_t bits = __ballot_sync(0xffffffffu, ok) & 0xffffu;
        if (lane == 0) s_bits[st] = bits;
        const uint32_t base = ring_s + st * 2 * C::kTile;
#pragma unroll
        for (int i = 0; i < kUnitTokens * CPR / 32; ++i) {
          const int x = i * 32 + lane, r = x / CPR, c = x % CPR;
          const bool in = c * 4 < a.dim;
          const int64_t o = __shfl_sync(0xffffffffu, off, r) + (in ? c * 4 : 0);
          const uint32_t bytes = in && ((bits >> r) & 1) ? 16 : 0;
          const uint32_t row = base + r * C::kRowBytes;
          cp_async16(row + ((c ^ (r & 7)) << 4), static_cast<const float*>(a.kc) + o, bytes);
          cp_async16(row + (c << 4) + C::kTile, static_cast<const float*>(a.vc) + o, bytes);
        }
        ++loaded;
        if (loaded < n) {
          cl.next(a);
          page = lane_page(a, cl, lane);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load();
    write_index<MR>(a, lane);

    const int t = lane & 15, hf = lane >> 4;
    float o[MR][VC], m[HR], l[HR];  // m, l: rows hf * HR + 0 .. HR - 1
    int lim[HR], first = 0, cut = 0;
    for (int it = 0; it < n; ++it) {
      __syncwarp();
      load();
      const int rows = cc.s.nq * a.group;
      if (it == 0 || cc.u == 0) {
        first = cc.u;
        if constexpr (kSeveral) cut = first_cut(a, cc);
#pragma unroll
        for (int r = 0; r < MR; ++r)
#pragma unroll
          for (int c = 0; c < VC; ++c) o[r][c] = 0.f;
#pragma unroll
        for (int e = 0; e < HR; ++e) {
          m[e] = WR_NEG_INF;
          l[e] = 0.f;
          lim[e] = row_limit(a, cc, (cc.rt * MR + hf * HR + e) / a.group);
        }
        for (int x = lane; x < MR * CPR; x += 32) {
          const int r = x / CPR, c = x % CPR, rr = cc.rt * MR + r, ii = rr / a.group;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (rr < rows && c * 4 < a.dim)
            v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) +
                                                 (int64_t)(cc.s.q0 + ii) * a.q_ts +
                                                 (int64_t)(cc.h * a.group + rr - ii * a.group) * a.q_hs +
                                                 c * 4);
          *reinterpret_cast<float4*>(qs + r * DP + c * 4) = v;
        }
      }
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const int st = it % kStages;
      const uint8_t* kb = ring + st * 2 * C::kTile;
      const uint8_t* vb = kb + C::kTile;
      const uint32_t bits = s_bits[st];
      float s[MR] = {};
      {
        const uint8_t* row = kb + t * C::kRowBytes;
#pragma unroll 4
        for (int c = 0; c < CPR / 2; ++c) {
          const int cc2 = hf * (CPR / 2) + c;
          const float4 k = *reinterpret_cast<const float4*>(row + ((cc2 ^ (t & 7)) << 4));
#pragma unroll
          for (int r = 0; r < MR; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(qs + r * DP + cc2 * 4);
            s[r] = fmaf(q.x, k.x, s[r]);
            s[r] = fmaf(q.y, k.y, s[r]);
            s[r] = fmaf(q.z, k.z, s[r]);
            s[r] = fmaf(q.w, k.w, s[r]);
          }
        }
      }
      // each half keeps its rows
      const int j = cc.u * kUnitTokens + t;
      const bool vis = (bits >> t) & 1;
      float x[HR], mx[HR];
      bool up = false;
#pragma unroll
      for (int e = 0; e < HR; ++e) {
        const float give = hf ? s[e] : s[e + HR], keep = hf ? s[e + HR] : s[e];
        const float sum = keep + __shfl_xor_sync(0xffffffffu, give, 16);
        x[e] = vis && j < lim[e] ? sum * a.scale_log2 : WR_NEG_INF;
        mx[e] = x[e];
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], d));
        up |= mx[e] > m[e];
      }
      if (__any_sync(0xffffffffu, up)) {
        float f[HR];
#pragma unroll
        for (int e = 0; e < HR; ++e) {
          const float nm = fmaxf(m[e], mx[e]);
          f[e] = nm == m[e] ? 1.f : ex2(m[e] - nm);
          m[e] = nm;
          l[e] *= f[e];
        }
#pragma unroll
        for (int r = 0; r < MR; ++r) {
          const float fr = __shfl_sync(0xffffffffu, f[r % HR], (r / HR) << 4);
#pragma unroll
          for (int c = 0; c < VC; ++c) o[r][c] *= fr;
        }
      }
      bool odd = false;
      if (kSeveral && cc.u >= cut) {
        uint32_t x = 0;
        auto look = [&](uint32_t v) { x |= (v & 0x7f800000u) + 0x00800000u; };
#pragma unroll 4
        for (int i = lane; i < C::kTile / 16; i += 32) {
          const uint4 v = reinterpret_cast<const uint4*>(vb)[i];
          look(v.x); look(v.y); look(v.z); look(v.w);
        }
        odd = __any_sync(0xffffffffu, x >> 31);
      }
#pragma unroll
      for (int e = 0; e < HR; ++e) {
        const float w = ex2(x[e] - (m[e] == WR_NEG_INF ? 0.f : m[e]));
        l[e] += w;
        ps[t * MR + hf * HR + e] = odd && j >= lim[e] ? -1.f : w;  // below zero: not seen
      }
      __syncwarp();
      auto key = [&](int k, auto seen) {
        float p[MR];
#pragma unroll
        for (int r = 0; r < MR; r += 4)
          *reinterpret_cast<float4*>(p + r) = *reinterpret_cast<const float4*>(ps + k * MR + r);
        float v[VC];
#pragma unroll
        for (int g = 0; g < VC; g += VW) {
          const uint8_t* src = vb + k * C::kRowBytes + (g * 32 + lane * VW) * 4;
          if constexpr (VW == 4) {
            const float4 f = *reinterpret_cast<const float4*>(src);
            v[g] = f.x; v[g + 1] = f.y; v[g + 2] = f.z; v[g + 3] = f.w;
          } else {
            const float2 f = *reinterpret_cast<const float2*>(src);
            v[g] = f.x; v[g + 1] = f.y;
          }
        }
#pragma unroll
        for (int r = 0; r < MR; ++r)
          if (seen(p[r]))
#pragma unroll
            for (int c = 0; c < VC; ++c) o[r][c] = fmaf(p[r], v[c], o[r][c]);
      };
      if (!odd) {
#pragma unroll 4
        for (int k = 0; k < kUnitTokens; ++k) key(k, [](float) { return true; });
      } else {
#pragma unroll 1
        for (int k = 0; k < kUnitTokens; ++k) key(k, [](float w) { return !(w < 0.f); });
      }
      const bool tile_end = cc.u == cc.us - 1;
      if (tile_end || it == n - 1) {
        float ls[HR];
#pragma unroll
        for (int e = 0; e < HR; ++e) {
          ls[e] = l[e];
#pragma unroll
          for (int d = 1; d < 16; d <<= 1) ls[e] += __shfl_xor_sync(0xffffffffu, ls[e], d);
        }
        const bool whole = tile_end && first == 0, lead = a.lead > 0 && cc.b == 0;
#pragma unroll
        for (int r = 0; r < MR; ++r) {
          const float mm = __shfl_sync(0xffffffffu, m[r % HR], (r / HR) << 4);
          const float ll = __shfl_sync(0xffffffffu, ls[r % HR], (r / HR) << 4);
          const int rr = cc.rt * MR + r;
          if (rr >= rows) continue;
          const int i = rr / a.group;
          const int64_t orow = (int64_t)(cc.s.q0 + i) * a.hq + cc.h * a.group + (rr - i * a.group);
          const int64_t prow = (w * 2 + (first == 0 ? 1 : 0)) * MR + r;
          const bool fin = whole && a.direct;
          const float inv = !fin ? 1.f : (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll));
          float* op = fin ? static_cast<float*>(a.out) + orow * a.dim
                          : (!whole ? a.part.piece + prow * a.dim : (lead ? a.lead_home : a.home) + orow * a.dim);
#pragma unroll
          for (int g = 0; g < VC; g += VW) {
            const int d = g * 32 + lane * VW;
            if (d < a.dim)
#pragma unroll
              for (int c = 0; c < VW; ++c) op[d + c] = o[r][g + c] * inv;
          }
          if (lane == 0) {
            if (!fin) *(!whole ? a.part.piece_ml + prow : (lead ? a.lead_home_ml : a.home_ml) + orow) = make_float2(mm, ll);
            else if (a.lse) a.lse[orow] = ll == 0.f ? WR_NEG_INF : (mm + log2f(ll)) * kLn2;
          }
        }
      }
      if (it + 1 < n) cc.next(a);
    }
    cp_async_wait<0>();
    if (kSeveral && a.ends && lane == 0)
      a.ends[w] = make_int4(cc.b, cc.h, cc.rt, cc.u == cc.us - 1 || first > 0 ? -1 : cc.u);
  } else {
    write_index<MR>(a, lane);
  }
  griddep_wait();
}

// ---------------------------------------------------------------------------
// Joining the pieces
// ---------------------------------------------------------------------------
struct CombineArgs {
  AttnArgs own;       // the launch of k_attn_stream*
  int64_t own_warps;
  int has_pre;        // the prefix's partial results: of that launch's segment 0,
                      // or of the tensor cores' launch,
  int tiles;          // then with this split and these rows a tile, tiles a key
  AttnPartials pre;   // head and units of its keys
  const float* pre_home;
  const float2* pre_home_ml;
  AttnSplit pre_split;
  int pre_mr, pre_rts, pre_us;
};

// A row's pieces of one launch: whole (in home), or n in slots of the warps
// (or CTAs) from w0 on.
struct PieceList {
  int64_t w0;
  int n, rl;
  bool whole;
};
WR_DEVINL PieceList piece_list(const AttnSplit& sp, int64_t unit0, int us, int row_in_tile) {
  PieceList p;
  const int64_t w0 = range_of(sp, unit0), w1 = range_of(sp, unit0 + us - 1);
  p.whole = w0 == w1;
  p.w0 = w0;
  p.n = (int)(w1 - w0) + 1;
  p.rl = row_in_tile;
  return p;
}

// A row's pieces lo .. hi - 1, 32 at a time: lane i looks up piece i and its
// weight, then all lanes add up the pieces' columns.  The loads of the first
// few pieces are under way before any weight is known (the pieces have often
// left L2 by now: one wait for HBM, not two).
template <int MR, int DP>
struct RowSum {
  static constexpr int VC = DP / 32, VW = VC < 4 ? VC : 4;  // columns a lane has, in runs of VW
  static constexpr int kFlight = DP > 128 ? 2 : 4;
  float m, l, o[VC];

  WR_DEVINL void add(const CombineArgs& c, const PieceList& po, const PieceList& pp, int64_t row, int lo, int hi,
                     int lane) {
    const AttnArgs& a = c.own;
    m = WR_NEG_INF;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < VC; ++i) o[i] = 0.f;
    for (int c0 = lo; c0 < hi; c0 += 32) {
      const int i = c0 + lane;
      const float* src = nullptr;
      float2 ml = make_float2(WR_NEG_INF, 0.f);
      if (i < hi) {
        const bool mine = i < po.n;
        const PieceList& p = mine ? po : pp;
        const int k = mine ? i : i - po.n;
        const int64_t at = p.whole ? row : ((p.w0 + k) * 2 + (k == 0 ? 1 : 0)) * (mine ? MR : c.pre_mr) + p.rl;
        src = (p.whole ? (mine ? a.home : c.pre_home) : (mine ? a.part.piece : c.pre.piece)) + at * a.dim;
        ml = (p.whole ? (mine ? a.home_ml : c.pre_home_ml) : (mine ? a.part.piece_ml : c.pre.piece_ml))[at];
      }
      const int n = min(32, hi - c0);
      float v[kFlight][VC];
      auto fetch = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          const float* p = reinterpret_cast<const float*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), min(k0 + k, n - 1)));
#pragma unroll
          for (int q = 0; q < VC; q += VW) {
            const int d = q * 32 + lane * VW;
            const bool in = d < a.dim && k0 + k < n;
            if constexpr (VW == 4) {
              const float4 x = in ? *reinterpret_cast<const float4*>(p + d) : make_float4(0.f, 0.f, 0.f, 0.f);
              v[k][q] = x.x; v[k][q + 1] = x.y; v[k][q + 2] = x.z; v[k][q + 3] = x.w;
            } else {
              const float2 x = in ? *reinterpret_cast<const float2*>(p + d) : make_float2(0.f, 0.f);
              v[k][q] = x.x; v[k][q + 1] = x.y;
            }
          }
        }
      };
      fetch(0);
      float nm = fmaxf(m, ml.x);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, d));
      const float base = nm == WR_NEG_INF ? 0.f : nm;
      const float fo = ex2(m - base), w = ex2(ml.x - base);
      float add = ml.y * w;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
      m = nm;
      l = l * fo + add;
#pragma unroll
      for (int q = 0; q < VC; ++q) o[q] *= fo;
#pragma unroll 1
      for (int k0 = 0;;) {
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          const float f = __shfl_sync(0xffffffffu, w, min(k0 + k, n - 1));
          if (k0 + k < n)
#pragma unroll
            for (int q = 0; q < VC; ++q) o[q] += f * v[k][q];
        }
        k0 += kFlight;
        if (k0 >= n) break;
        fetch(k0);
      }
    }
  }

  template <typename T>
  WR_DEVINL void store(const AttnArgs& a, int64_t row, int lane) const {
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
#pragma unroll
    for (int q = 0; q < VC; q += VW) {
      const int d = q * 32 + lane * VW;
      if (d >= a.dim) continue;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < VW; e += 2)
          *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row * a.dim + d + e) =
              pack_bf16(o[q + e] * inv, o[q + e + 1] * inv);
      } else {
#pragma unroll
        for (int e = 0; e < VW; ++e) static_cast<float*>(a.out)[row * a.dim + d + e] = o[q + e] * inv;
      }
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? WR_NEG_INF : (m + log2f(l)) * kLn2;
  }
};

// The pieces of row g of token t and key head h.
struct RowPlace {
  Segment s;
  int us, rts;
  int64_t unit0;
  AttnSplit sp;
};
template <int MR>
WR_DEVINL bool row_pieces(const CombineArgs& c, const RowPlace& x, int t, int h, int g, PieceList& po, PieceList& pp) {
  const AttnArgs& a = c.own;
  const int r = (t - x.s.q0) * a.group + g;
  po = piece_list(x.sp, x.unit0 + ((int64_t)h * x.rts + r / MR) * x.us, x.us, r % MR);
  if (po.whole && a.direct) return false;  // written by the first kernel
  if (c.has_pre) {
    const int rp = t * a.group + g, rt = rp / c.pre_mr;
    pp = piece_list(c.tiles ? c.pre_split : x.sp, ((int64_t)h * c.pre_rts + rt) * c.pre_us, c.pre_us,
                    rp - rt * c.pre_mr);
  }
  return true;
}

// Few rows with many pieces: a CTA a row, each of its 8 warps an eighth of the
// pieces.  Where they are it works out from the lengths while the kernels
// before are still at it.
template <typename T, int MR, int DP>
__global__ void __launch_bounds__(256) k_attn_combine_wide(const CombineArgs c) {
  using R = RowSum<MR, DP>;
  constexpr int kWarps = 8;
  __shared__ float s_o[kWarps][DP];
  __shared__ float2 s_ml[kWarps];
  const AttnArgs& a = c.own;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int t = (int)row / a.hq, hq = (int)row - t * a.hq;
  const int h = hq / a.group, g = hq - h * a.group;
  RowPlace x{};
  const int b = a.q_start ? seq_of(a, t) : t, seg = b + (a.lead > 0);
  for (int i0 = 0; i0 < segments(a); i0 += 32) {
    const int64_t v = seg_units<MR>(a, i0 + lane);
    x.sp.units += v;
    if (i0 + lane < seg) x.unit0 += v;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    x.unit0 += __shfl_xor_sync(0xffffffffu, x.unit0, d);
    x.sp.units += __shfl_xor_sync(0xffffffffu, x.sp.units, d);
  }
  x.sp.ranges = min(c.own_warps, x.sp.units);
  PieceList po{}, pp{};
  bool work = true;
  if (b >= 0) {
    x.s = segment(a, seg);
    x.us = key_units(x.s);
    x.rts = row_tiles<MR>(a, x.s);
    work = row_pieces<MR>(c, x, t, h, g, po, pp);
  }
  griddep_wait();
  if (!work) return;
  const int total = po.n + pp.n;
  R sum;
  sum.add(c, po, pp, row, total * wid / kWarps, total * (wid + 1) / kWarps, lane);
#pragma unroll
  for (int q = 0; q < R::VC; q += R::VW)
#pragma unroll
    for (int e = 0; e < R::VW; ++e) s_o[wid][q * 32 + lane * R::VW + e] = sum.o[q + e];
  if (lane == 0) s_ml[wid] = make_float2(sum.m, sum.l);
  __syncthreads();
  if (wid) return;
  sum.m = WR_NEG_INF;
  for (int i = 0; i < kWarps; ++i) sum.m = fmaxf(sum.m, s_ml[i].x);
  const float base = sum.m == WR_NEG_INF ? 0.f : sum.m;
  sum.l = 0.f;
#pragma unroll
  for (int q = 0; q < R::VC; ++q) sum.o[q] = 0.f;
  for (int i = 0; i < kWarps; ++i) {
    const float f = ex2(s_ml[i].x - base);
    sum.l += s_ml[i].y * f;
#pragma unroll
    for (int q = 0; q < R::VC; q += R::VW)
#pragma unroll
      for (int e = 0; e < R::VW; ++e) sum.o[q + e] += s_o[i][q * 32 + lane * R::VW + e] * f;
  }
  sum.template store<T>(a, row, lane);
}

// Many rows: a warp a row.
template <typename T, int MR, int DP>
__global__ void __launch_bounds__(128) k_attn_combine(const CombineArgs c) {
  const AttnArgs& a = c.own;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  griddep_wait();
  if (row >= (int64_t)a.T * a.hq) return;
  const int t = (int)row / a.hq, hq = (int)row - t * a.hq;
  const int h = hq / a.group, g = hq - h * a.group;
  const int b = a.q_start ? a.token_seq[t] : t;
  PieceList po{}, pp{};
  if (b >= 0) {
    RowPlace x;
    x.unit0 = a.seg_unit[b + (a.lead > 0)];
    x.sp.units = a.seg_unit[segments(a)];
    x.sp.ranges = min(c.own_warps, x.sp.units);
    x.s = segment(a, b + (a.lead > 0));
    x.us = key_units(x.s);
    x.rts = row_tiles<MR>(a, x.s);
    if (!row_pieces<MR>(c, x, t, h, g, po, pp)) return;
  }
  RowSum<MR, DP> sum;
  sum.add(c, po, pp, row, 0, po.n + pp.n, lane);
  sum.template store<T>(a, row, lane);
}

// More rows than the warps of a launch can leave unfinished, and no prefix
// beside them: a warp a row of the tiles that a range's end cuts (209
// sequences of 1 to 64 tokens, their own keys and 64 heads of 96 columns: 13 us
// behind the first kernel's 244, and 126 with a look at every row).  The warp
// whose range begins a tile names it.  Only calls with several tokens a
// sequence have that many rows to make up for the naming (12 sequences of one
// token, 16 heads, fp32: 37.1 us without, 39.2 with).
template <typename T, int MR, int DP>
__global__ void __launch_bounds__(128) k_attn_combine_ends(const CombineArgs c) {
  const AttnArgs& a = c.own;
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), w = at / MR;
  const int rl = (int)(at % MR);
  griddep_wait();
  RowSum<MR, DP> sum;
  if (a.q_start)
    for (int64_t t = at; t < a.T; t += (int64_t)gridDim.x * 4)
      if (a.token_seq[t] < 0)
        for (int h = 0; h < a.hq; ++h) {
          sum.add(c, PieceList{}, PieceList{}, t * a.hq + h, 0, 0, lane);
          sum.template store<T>(a, t * a.hq + h, lane);
        }
  AttnSplit sp;
  sp.units = a.seg_unit[segments(a)];
  sp.ranges = min(c.own_warps, sp.units);
  if (w >= sp.ranges) return;
  const int4 e = a.ends[w];
  if (e.w < 0) return;
  const Segment s = segment(a, e.x);
  const int r = e.z * MR + rl, i = r / a.group;
  if (i >= s.nq) return;
  const int64_t row = (int64_t)(s.q0 + i) * a.hq + e.y * a.group + (r - i * a.group);
  const PieceList po = piece_list(sp, range_start(sp, w + 1) - 1 - e.w, key_units(s), rl);
  sum.add(c, po, PieceList{}, row, 0, po.n, lane);
  sum.template store<T>(a, row, lane);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// The prefix goes to the tensor cores from 33 rows a key head where the warps
// of k_attn_stream, which read the keys again for every 16 rows, would read
// more than this: below, that kernel's launch and set-up cost more.  Whole
// calls, us, without / with it, by the MB read so (8 key heads, 4 query heads
// each, 200 own keys a sequence, caches that are not in L2):
//   head  rows        16           34           64           128          256
//    64     64   15.8 / 19.7  18.7 / 21.3  23.4 / 24.5  34.2 / 30.3  53.7 / 40.3
//    64    256   20.3 / 23.7  24.4 / 31.2  28.6 / 29.8  39.4 / 32.7  58.4 / 39.0
//   128     64   15.4 / 22.1  18.1 / 22.8  23.1 / 24.8  32.0 / 30.5  50.1 / 38.4
//   128    128   21.2 / 27.1  23.7 / 32.9  27.7 / 28.8  37.2 / 30.9  55.1 / 38.3
//   128    256   24.1 / 30.8  26.4 / 36.3  29.8 / 33.3  38.9 / 37.2  57.4 / 41.3
//   128   1024   56.8 / 68.8  56.6 / 66.6  60.4 / 65.0  67.7 / 67.9  84.2 / 79.2
constexpr int kTileMinRows = 32;
constexpr int64_t kTileMinBytes = 64 << 20;

struct Plan {
  int dp, mr, smem;
  int own_grid, tile_grid;
  int inline_prefix; // each sequence reads the prefix with its own keys
  int has_pre;       // the prefix is a segment of its own,
  int tiles;         // on the tensor cores
  int tile_mr;
  int64_t rows;      // T * hq: of the output
  int ends;          // the join takes the tiles that the ranges' ends cut, not all rows
  size_t off_piece, off_piece_ml, off_home, off_home_ml, off_seg, off_tok, off_ends;
  size_t off_tpiece, off_tpiece_ml, off_phome, off_phome_ml;
  size_t bytes;
};

// Shared memory and rows a warp of the kernel that takes this problem.
void kernel_shape(const AttnProblem& p, Plan* pl) {
  pl->dp = p.c.dim <= 64 ? 64 : (p.c.dim <= 128 ? 128 : 256);
  if (p.c.dtype != WR_DTYPE_F32) {
    pl->mr = 16;
    pl->smem = pl->dp == 64 ? StreamCfg<64>::kSmem : pl->dp == 128 ? StreamCfg<128>::kSmem : StreamCfg<256>::kSmem;
    return;
  }
  // 8 rows a warp where the sequences have more than 4 (twice the products
  // for a key read); a sequence with 1 row wastes 3 of 4 rather than 7 of 8.
  pl->mr = (int64_t)p.T * (p.hq / p.c.hkv) > 4 * (int64_t)p.B ? 8 : 4;
  if (pl->mr == 8)
    pl->smem = pl->dp == 64 ? StreamF32Cfg<64, 8>::kSmem : pl->dp == 128 ? StreamF32Cfg<128, 8>::kSmem
                                                                          : StreamF32Cfg<256, 8>::kSmem;
  else
    pl->smem = pl->dp == 64 ? StreamF32Cfg<64, 4>::kSmem : pl->dp == 128 ? StreamF32Cfg<128, 4>::kSmem
                                                                          : StreamF32Cfg<256, 4>::kSmem;
}

Plan make_plan(const AttnProblem& p) {
  Plan pl{};
  kernel_shape(p, &pl);
  const int fit = 227 * 1024 / (pl.smem + 2048);
  const int per_sm = fit < 1 ? 1 : (fit > 16 ? 16 : fit);
  const int64_t most = (int64_t)device_sm_count() * per_sm;
  const int group = p.hq / p.c.hkv;
  pl.rows = (int64_t)p.T * p.hq;
  pl.inline_prefix = p.prefix_len > 0 && p.B == 1;
  pl.has_pre = p.prefix_len > 0 && !pl.inline_prefix;
  const int64_t group_rows = (int64_t)p.T * group;  // rows that meet the prefix, a key head
  const int64_t again = (group_rows + 15) / 16 * p.c.hkv * p.prefix_len * p.c.dim * 4;  // K and V in bf16
  pl.tiles = pl.has_pre && group_rows > kTileMinRows && again > kTileMinBytes && prefix_tiles_ok(p);
  // An upper bound of the units: the lengths are on the device.
  const int64_t keys = (int64_t)p.table_width * p.c.page_size + (pl.inline_prefix ? p.prefix_len : 0);
  const int64_t tiles = (group_rows + pl.mr - 1) / pl.mr + (p.B > 0 ? p.B : 0);
  int64_t units = (tiles * p.c.hkv) * ((keys + kUnitTokens - 1) / kUnitTokens + 1);
  if (pl.has_pre && !pl.tiles) units += tiles * p.c.hkv * ((p.prefix_len + kUnitTokens - 1) / kUnitTokens);
  pl.own_grid = (int)(units < most ? (units < 1 ? 1 : units) : most);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += (n + 255) & ~(size_t)255;
    return o;
  };
  const size_t own_rows = (size_t)pl.own_grid * 2 * pl.mr;
  pl.off_piece = take(own_rows * p.c.dim * 4);
  pl.off_piece_ml = take(own_rows * 8);
  pl.off_seg = take((size_t)(p.B + 2) * 8);
  pl.off_tok = take((size_t)(p.q_start ? p.T : 0) * 4);
  pl.ends = p.q_start && !pl.has_pre && pl.rows > (int64_t)pl.own_grid * pl.mr;
  pl.off_ends = take(pl.ends ? (size_t)pl.own_grid * 16 : 0);
  if (pl.has_pre) {
    pl.off_home = take((size_t)pl.rows * p.c.dim * 4);
    pl.off_home_ml = take((size_t)pl.rows * 8);
    pl.off_phome = take((size_t)pl.rows * p.c.dim * 4);
    pl.off_phome_ml = take((size_t)pl.rows * 8);
  }
  if (pl.tiles) {
    pl.tile_mr = group_rows > 128 ? 256 : 128;
    const int64_t tu = (int64_t)p.c.hkv * ((group_rows + pl.tile_mr - 1) / pl.tile_mr) *
                       ((p.prefix_len + kPrefixUnit - 1) / kPrefixUnit);
    pl.tile_grid = (int)(tu < device_sm_count() ? tu : device_sm_count());
    const size_t tile_rows = (size_t)pl.tile_grid * 2 * pl.tile_mr;
    pl.off_tpiece = take(tile_rows * p.c.dim * 4);
    pl.off_tpiece_ml = take(tile_rows * 8);
  }
  pl.bytes = at;
  return pl;
}

template <typename K>
cudaError_t launch_one(K kernel, int64_t grid, int threads, int smem, bool pdl, cudaStream_t stream,
                       const void* args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  void* ptrs[1] = {const_cast<void*>(args)};
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), ptrs);
}

template <bool kSeveral>
cudaError_t launch_stream(const Plan& pl, bool f32, const AttnArgs& a, cudaStream_t s) {
  auto go = [&](auto kernel) { return launch_one(kernel, pl.own_grid, 32, pl.smem, false, s, &a); };
  if (f32 && pl.mr == 8)
    return pl.dp == 64    ? go(k_attn_stream_f32<64, 8, kSeveral>)
           : pl.dp == 128 ? go(k_attn_stream_f32<128, 8, kSeveral>)
                          : go(k_attn_stream_f32<256, 8, kSeveral>);
  if (f32)
    return pl.dp == 64    ? go(k_attn_stream_f32<64, 4, kSeveral>)
           : pl.dp == 128 ? go(k_attn_stream_f32<128, 4, kSeveral>)
                          : go(k_attn_stream_f32<256, 4, kSeveral>);
  return pl.dp == 64    ? go(k_attn_stream<64, kSeveral>)
         : pl.dp == 128 ? go(k_attn_stream<128, kSeveral>)
                        : go(k_attn_stream<256, kSeveral>);
}

template <typename T, int MR>
cudaError_t launch_combine(int dp, const CombineArgs& c, cudaStream_t s) {
  const int64_t rows = (int64_t)c.own.T * c.own.hq;
  if (c.own.ends) {
    auto go = [&](auto kernel) { return launch_one(kernel, c.own_warps * MR / 4, 128, 0, true, s, &c); };
    return dp == 64 ? go(k_attn_combine_ends<T, MR, 64>) : dp == 128 ? go(k_attn_combine_ends<T, MR, 128>)
                                                                     : go(k_attn_combine_ends<T, MR, 256>);
  }
  if (rows <= (int64_t)device_sm_count() * 8) {
    auto go = [&](auto kernel) { return launch_one(kernel, rows, 256, 0, true, s, &c); };
    return dp == 64 ? go(k_attn_combine_wide<T, MR, 64>) : dp == 128 ? go(k_attn_combine_wide<T, MR, 128>)
                                                                     : go(k_attn_combine_wide<T, MR, 256>);
  }
  auto go = [&](auto kernel) { return launch_one(kernel, (rows + 3) / 4, 128, 0, true, s, &c); };
  return dp == 64 ? go(k_attn_combine<T, MR, 64>) : dp == 128 ? go(k_attn_combine<T, MR, 128>)
                                                              : go(k_attn_combine<T, MR, 256>);
}

}  // namespace

size_t attn_workspace_bytes(const AttnProblem& p) { return make_plan(p).bytes; }

wr_status_t launch_attn(const AttnProblem& p, void* ws, cudaStream_t stream) {
  const Plan pl = make_plan(p);
  const bool f32 = p.c.dtype == WR_DTYPE_F32;
  uint8_t* base = static_cast<uint8_t*>(ws);
  AttnArgs a{};
  a.q = p.q; a.kc = p.c.k; a.vc = p.c.v;
  a.q_ts = p.q_ts; a.q_hs = p.q_hs;
  a.page_stride = p.c.page_stride; a.head_stride = p.c.head_stride; a.slot_stride = p.c.slot_stride;
  a.tables = p.tables; a.table_stride = p.table_stride; a.lens = p.lens; a.q_start = p.q_start;
  a.prefix_pages = p.prefix_pages;
  a.num_pages = p.c.num_pages; a.page_size = p.c.page_size;
  a.page_shift = (p.c.page_size & (p.c.page_size - 1)) == 0 ? __builtin_ctz(p.c.page_size) : -1;
  a.T = p.T; a.B = p.B; a.hq = p.hq; a.hkv = p.c.hkv; a.group = p.hq / p.c.hkv; a.dim = p.c.dim;
  a.table_width = p.table_width;
  a.prefix = pl.inline_prefix ? p.prefix_len : 0;
  a.lead = pl.has_pre && !pl.tiles ? p.prefix_len : 0;
  a.direct = !pl.has_pre;
  a.scale_log2 = p.scale * kLog2e;
  a.part.piece = reinterpret_cast<float*>(base + pl.off_piece);
  a.part.piece_ml = reinterpret_cast<float2*>(base + pl.off_piece_ml);
  a.home = reinterpret_cast<float*>(base + pl.off_home);
  a.home_ml = reinterpret_cast<float2*>(base + pl.off_home_ml);
  a.lead_home = reinterpret_cast<float*>(base + pl.off_phome);
  a.lead_home_ml = reinterpret_cast<float2*>(base + pl.off_phome_ml);
  a.seg_unit = reinterpret_cast<int64_t*>(base + pl.off_seg);
  a.token_seq = reinterpret_cast<int32_t*>(base + pl.off_tok);
  a.ends = pl.ends ? reinterpret_cast<int4*>(base + pl.off_ends) : nullptr;
  a.out = p.out; a.lse = p.lse;
  CombineArgs c{};
  c.own = a;
  c.own_warps = pl.own_grid;
  if (pl.has_pre) {
    c.has_pre = 1;
    c.tiles = pl.tiles;
    c.pre = a.part;
    c.pre_home = a.lead_home;
    c.pre_home_ml = a.lead_home_ml;
    c.pre_mr = pl.tiles ? pl.tile_mr : pl.mr;
    const int unit = pl.tiles ? kPrefixUnit : kUnitTokens;
    c.pre_rts = (int)(((int64_t)p.T * a.group + c.pre_mr - 1) / c.pre_mr);
    c.pre_us = (p.prefix_len + unit - 1) / unit;
  }
  // With one token a sequence the look for values that are not finite falls
  // away (12 sequences, 16 heads, fp32: 37 us without it, 41 with).
  cudaError_t e = p.q_start ? launch_stream<true>(pl, f32, a, stream) : launch_stream<false>(pl, f32, a, stream);
  if (e != cudaSuccess) return cuda_fail(e, "shared_prefix_attention launch");
  if (pl.tiles) {
    // After the own keys, so that the prefix's partial results, the larger
    // part, are still in L2 when they are joined.
    AttnArgs x = a;
    x.prefix = p.prefix_len;
    x.part.piece = reinterpret_cast<float*>(base + pl.off_tpiece);
    x.part.piece_ml = reinterpret_cast<float2*>(base + pl.off_tpiece_ml);
    x.home = a.lead_home;
    x.home_ml = a.lead_home_ml;
    c.pre = x.part;
    c.pre_split.units = (int64_t)a.hkv * c.pre_rts * c.pre_us;
    c.pre_split.ranges = pl.tile_grid < c.pre_split.units ? pl.tile_grid : c.pre_split.units;
    const wr_status_t st = launch_attn_prefix(p, x, pl.tile_mr, pl.tile_grid, stream);
    if (st != WR_OK) return st;
  }
  e = !f32 ? launch_combine<uint16_t, 16>(pl.dp, c, stream)
           : pl.mr == 8 ? launch_combine<float, 8>(pl.dp, c, stream) : launch_combine<float, 4>(pl.dp, c, stream);
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "shared_prefix_attention (join) launch");
}

}  // namespace wr
