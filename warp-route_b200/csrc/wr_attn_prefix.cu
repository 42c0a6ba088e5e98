// wr_attn_prefix.cu — the shared prefix's part of the attention on the tensor
// cores: the rows of all sequences' tokens meet the prefix's keys once.
//
// A product of [rows, keys] and one of [rows, dim], 4 * rows * keys * dim
// operations for 4 * keys * dim bytes: from some 200 rows a key head on the
// tensor cores (and, next to them, the exponentials: rows * keys of them, 16 a
// cycle and SM, take as long as both products at dim 128) bound it, below that
// HBM.
//
// A CTA has one SM and NT tiles of 128 rows (NT 2 when there are that many:
// while one tile's softmax runs, the tensor core works on the other).  Per
// 64 keys: S = Q K^T into TMEM; a thread reads its row of S (lane = row, so
// no exchange between threads), takes the running maximum and the weights
// 2^(s - m), which go back over S as bf16, the A operand of O += P V, whose
// sum stays in TMEM for all of a piece's keys.  S has two buffers of 64
// columns a tile (with O of both tiles TMEM is full), so the next scores are
// there when a softmax ends; with one of 128 columns, whose P has to be
// consumed before the next S, softmax and products of a tile took turns
// (145 us for 1536 rows and 16384 keys of 8 heads; now 100 us, 1.05 PFLOP/s, at
// the 1.5 GHz that the power limit leaves, and 2 us more for the votes on waits).  m follows the true maximum
// only when it has grown by more than 8 (a factor of 256, harmless in fp32
// sums and bf16 weights), so O is rescaled rarely.  Warp 4 * NT brings K and V
// by TMA, a copy a page and 64 columns, into two rings; the warps behind it
// issue the MMAs, for each tile one the scores' and one the sums'.  Keys in
// pages outside the cache, and those behind the prefix's end in its last page,
// are masked in S and their rows of V set to zero.
//
// The (key head, row tiles, 128 keys) units are dealt to the CTAs in ranges of
// equal length, their pieces joined by k_attn_combine (wr_attention.cu).
//
// Every wait is bounded.  One that runs out ends the CTA's work and leaves NaN
// in the rows of its pieces, in their sums, so that it shows in the output.
// Whether a wait ran out is one answer for all lanes of a warp (wait_warp),
// since what follows is done by whole warps (tcgen05.ld and st, votes, elect).
#include "wr_attention.cuh"
#include "wr_tcgen05.cuh"

namespace wr {
namespace {

constexpr int kTileKeys = kPrefixUnit;
constexpr int kTileRows = 128;
constexpr int kHalf = 64;  // keys of one S buffer
constexpr int kMaskRing = 8;
constexpr float kRescale = 8.f;
#define WR_NEG_INF (-__int_as_float(0x7f800000))

template <int D, int NT>
struct Cfg {
  static constexpr int kStages = D == 64 ? 4 : (NT == 2 ? 2 : 3);
  static_assert(kStages <= 4, "mask ring");
  static constexpr int kPanels = D / 64;
  static constexpr int kPanelBytes = 128 * 128;  // 128 rows of 64 columns
  static constexpr int kTileBytes = kPanels * kPanelBytes;
  static constexpr int kSmem = 1024 + NT * kTileBytes + 2 * kStages * kTileBytes;
  static constexpr int kThreads = NT * 128 + 32 + NT * 64;
  static constexpr uint32_t kTmemCols = NT == 2 ? 512 : 256;
};

struct PrefixArgs {
  AttnArgs a;
  int pairs;  // row tiles of NT * 128 rows a key head
  int us;     // units of 128 keys
  AttnSplit sp;
  int box;    // keys of one TMA copy
  uint32_t group_inv;  // ceil(2^32 / group), 0 for a group of one
};

// Token of a row: its quotient by the group, exact while row * group < 2^32.
WR_DEVINL int token_of(const PrefixArgs& p, int row) {
  return p.group_inv ? (int)__umulhi((uint32_t)row, p.group_inv) : row;
}

WR_DEVINL float ex2p(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Bound of the waits that the work hangs on, in ns; with 0 each gives up at
// once.  The waits for what is still in flight when a CTA ends are not among
// them: those always have the whole kWaitLimitNs.
#ifndef WR_PREFIX_WAIT_NS
#define WR_PREFIX_WAIT_NS kWaitLimitNs
#endif
constexpr uint64_t kPrefixWaitNs = WR_PREFIX_WAIT_NS;

// A wait of a whole converged warp: few instructions (the MMA warps spend
// their time on them), each try suspended by the hardware; the clock comes in
// only when many have failed.  False, for all lanes: it gave up, or another
// warp had.  (The vote costs 1 % of a call bound by this kernel: 191.1 us
// without, 193.0 with, for 256 sequences of 6 rows a key head behind 16384
// keys.)
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  return mbar_wait(bar, parity, abort, kPrefixWaitNs);
}
WR_DEVINL bool wait_warp(uint64_t* bar, uint32_t parity, const volatile int* abort = nullptr) {
  if (kPrefixWaitNs == 0) return false;
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 200;\n\t"
      "WAIT_%=:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "@P bra DONE_%=;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 P, n, 0;\n\t"
      "@P bra WAIT_%=;\n\t"
      "DONE_%=:\n\t"
      "min.u32 %0, n, 1;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, ok != 0 || wait_long(bar, parity, abort));
}

// A CTA's pieces in order: the units of one (key head, row tiles) in its range.
struct Piece {
  int h, pair, u, n;
};
WR_DEVINL Piece piece_at(const PrefixArgs& p, int64_t unit, int64_t end) {
  Piece x;
  const int64_t tile = quotient(unit, p.us);
  x.u = (int)(unit - tile * p.us);
  x.h = (int)quotient(tile, p.pairs);
  x.pair = (int)(tile - (int64_t)x.h * p.pairs);
  x.n = (int)min((int64_t)(p.us - x.u), end - unit);
  return x;
}

template <int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::kThreads, 1)
    k_attn_prefix(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  const PrefixArgs p) {
  using C = Cfg<D, NT>;
  constexpr int S = C::kStages, MR = NT * kTileRows;
  extern __shared__ uint8_t s_raw[];
  __shared__ uint64_t k_full[S], k_empty[S], v_full[S], v_empty[S], aux;
  __shared__ uint64_t q_full[NT], s_full[NT][2], p_full[NT][2], pv_done[NT][2], turn[NT], drain[2 * NT];
  __shared__ uint32_t s_mask[kMaskRing][4], s_special[kMaskRing], s_tmem;
  __shared__ int s_abort;
  const AttnArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qbuf = smem;
  uint8_t* kbuf = qbuf + NT * C::kTileBytes;
  uint8_t* vbuf = kbuf + S * C::kTileBytes;
  volatile int* abort = &s_abort;

  griddep_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], NT);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], NT);
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&q_full[t], kTileRows);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[t][b], 1);
        mbar_init(&p_full[t][b], kTileRows);
        mbar_init(&pv_done[t][b], 1);
      }
      mbar_init(&drain[t], 1);
      mbar_init(&drain[NT + t], 1);
      mbar_init(&turn[t], 4);
    }
    mbar_init(&aux, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == NT * 4 + 1) {
    tmem_alloc(&s_tmem, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t tmem_s = tmem, tmem_o = tmem + NT * kTileKeys;
  const int64_t u0 = range_start(p.sp, blockIdx.x), u1 = range_start(p.sp, blockIdx.x + 1);
  const int total = (int)(u1 - u0);

  if (warp == NT * 4) {
    // ---- K and V, by TMA -------------------------------------------------
    const uint64_t policy = l2_policy_evict_last();  // other CTAs read the same keys
    const int per_tile = kTileKeys / p.box;          // copies a tile and panel
    const int ops = per_tile * C::kPanels;
    const uint32_t op_bytes = (uint32_t)p.box * 128;
    int issued_k = 0, issued_v = 0;
    uint32_t aux_phase = 0;
    int64_t unit = u0;
    int it = 0;
    bool dead = false;  // this warp or another gave up
    while (it < total && !dead) {
      const Piece pc = piece_at(p, unit, u1);
      for (int i = 0; i < pc.n; ++i, ++it) {
        const int st = it % S;
        const uint32_t ph = (it / S) & 1;
        const int key0 = (pc.u + i) * kTileKeys;
        const int pi = lane / C::kPanels, panel = lane % C::kPanels;
        const int k0 = key0 + pi * p.box;
        int page = -1, row = 0;
        if (lane < ops && k0 < a.prefix) {
          int idx;
          split_page(k0, a.page_size, a.page_shift, idx, row);
          page = __ldg(a.prefix_pages + idx);
        }
        const bool ok = page >= 0 && page < a.num_pages;
        const uint32_t oks = __ballot_sync(0xffffffffu, ok);
        const uint32_t bytes = __popc(oks) * op_bytes;
        const bool special = __popc(oks) != ops || key0 + kTileKeys > a.prefix;
        // Keys of this tile that count: word w of the mask, by lane w.
        uint32_t word = 0xffffffffu;
        if (special) {
          word = 0;
          for (int j = 0; j < 32; ++j) {
            const int key = lane * 32 + j;  // lanes 0..3 alone are used
            const bool in = lane < 4 && key0 + key < a.prefix && ((oks >> ((key / p.box) * C::kPanels)) & 1);
            word |= (uint32_t)in << j;
          }
        }
        dead = __any_sync(0xffffffffu, *abort) || (it >= S && !wait_warp(&k_empty[st], ph ^ 1, abort));
        if (dead) break;
        if (lane < 4) s_mask[it % kMaskRing][lane] = word;
        if (lane == 0) s_special[it % kMaskRing] = special;
        __syncwarp();
        if (lane == 0) {
          if (bytes) mbar_arrive_expect_tx(&k_full[st], bytes); else mbar_arrive(&k_full[st]);
        }
        __syncwarp();
        uint8_t* dst = kbuf + st * C::kTileBytes + panel * C::kPanelBytes + pi * p.box * 128;
        if (ok) tma_load_4d(dst, &kmap, panel * 64, row, pc.h, page, &k_full[st], policy);
        issued_k = it + 1;
        dead = it >= S && !wait_warp(&v_empty[st], ph ^ 1, abort);
        if (dead) break;
        dst += vbuf - kbuf;
        uint64_t* bar = special ? &aux : &v_full[st];
        if (lane == 0) {
          if (bytes) mbar_arrive_expect_tx(bar, bytes); else mbar_arrive(bar);
        }
        __syncwarp();
        if (ok) tma_load_4d(dst, &vmap, panel * 64, row, pc.h, page, bar, policy);
        if (special) {
          // What the copies left behind the prefix, or did not bring, becomes 0.
          // (Copies of this warp's: the whole limit.  Without them V never
          // becomes full, and the warps that wait for it give up too.)
          dead = !__all_sync(0xffffffffu, mbar_wait(&aux, aux_phase, nullptr));
          if (dead) break;
          aux_phase ^= 1;
          for (int key = 0; key < kTileKeys; ++key) {
            const uint32_t w = __shfl_sync(0xffffffffu, word, key >> 5);
            if ((w >> (key & 31)) & 1) continue;
            if (lane < 8 * C::kPanels)
              *reinterpret_cast<uint4*>(vbuf + st * C::kTileBytes + (lane >> 3) * C::kPanelBytes + key * 128 +
                                        (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
        }
        issued_v = it + 1;
      }
      unit += pc.n;
    }
    // Nothing of this CTA's is in flight when it ends: copies have landed, and
    // (unless it gave up) the MMAs have released the stages.
    if (dead) *abort = 1;
    dead = __any_sync(0xffffffffu, *abort);
    for (int i = max(0, issued_k - S); i < issued_k; ++i)
      mbar_wait(dead ? &k_full[i % S] : &k_empty[i % S], (i / S) & 1, nullptr);
    for (int i = max(0, issued_v - S); i < issued_v; ++i)
      mbar_wait(dead ? &v_full[i % S] : &v_empty[i % S], (i / S) & 1, nullptr);
  } else if (warp > NT * 4) {
    // ---- the MMAs ---------------------------------------------------------
    // A warp for each tile's scores and one for its sums: what one waits for
    // does not hold up the other.  S(j) needs K and, since P(j - 2) lies in its
    // columns, the end of PV(j - 2); PV(j) needs P(j) and V.  (j: half tiles of
    // this CTA, two in a stage.)  The whole warp walks through the loop and one
    // elected lane issues: the descriptors then stay in uniform registers,
    // where the MMAs want them (in a branch of one lane each takes a detour of
    // some 70 cycles).
    const int which = __shfl_sync(0xffffffffu, warp, 0) - NT * 4 - 1;
    const int t = which % NT;
    const uint32_t st = tmem_s + t * 2 * kHalf;
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) { dead |= !wait_warp(bar, parity); };
    int64_t unit = u0;
    int j = 0, piece = 0;
    if (which < NT) {  // S = Q K^T
      const uint32_t idesc = idesc_bf16(kTileRows, kHalf);
      const uint64_t qd = sw128_desc(smem_u32(qbuf + t * C::kTileBytes)), kd = sw128_desc(smem_u32(kbuf));
      while (j < 2 * total && !dead) {
        const Piece pc = piece_at(p, unit, u1);
        wait(&q_full[t], piece & 1);
        for (const int end = j + 2 * pc.n; j < end && !dead; ++j) {
          const int b = j & 1, it = j >> 1, stage = it % S;
          if (b == 0) wait(&k_full[stage], (it / S) & 1);
          if (j >= 2) wait(&pv_done[t][b], (it - 1) & 1);
          tc_fence_after();
          const uint64_t kk = kd + ((uint64_t)(stage * C::kTileBytes + b * kHalf * 128) >> 4);
          if (elect_one() && !dead) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint64_t ko = ((k >> 2) * C::kPanelBytes + (k & 3) * 32) >> 4;
              umma_bf16(st + b * kHalf, qd + ko, kk + ko, idesc, k > 0);
            }
            umma_commit(&s_full[t][b]);
            if (b == 1) umma_commit(&k_empty[stage]);
          }
          __syncwarp();
        }
        unit += pc.n;
        ++piece;
      }
    } else {  // O (+)= P V
      const uint32_t idesc = idesc_bf16(kTileRows, D) | kIdescBMajorMn, ot = tmem_o + t * D;
      const uint64_t vd = sw128_desc_mn(smem_u32(vbuf), C::kPanelBytes);
      while (j < 2 * total && !dead) {
        const Piece pc = piece_at(p, unit, u1);
        const int first = j;
        for (const int end = j + 2 * pc.n; j < end && !dead; ++j) {
          const int b = j & 1, it = j >> 1, stage = it % S;
          if (b == 0) wait(&v_full[stage], (it / S) & 1);
          wait(&p_full[t][b], it & 1);
          tc_fence_after();
          const uint64_t vv = vd + ((uint64_t)(stage * C::kTileBytes + b * kHalf * 128) >> 4);
          if (elect_one() && !dead) {
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k)
              umma_bf16_ta(ot, st + b * kHalf + k * 8, vv + (k * 2048 >> 4), idesc, j > first || k > 0);
            umma_commit(&pv_done[t][b]);
            if (b == 1) umma_commit(&v_empty[stage]);
          }
          __syncwarp();
        }
        unit += pc.n;
      }
    }
    if (dead) {  // let what was issued end
      *abort = 1;
      if (elect_one()) umma_commit(&drain[which]);
      __syncwarp();
      mbar_wait(&drain[which], 0, nullptr);
    }
  } else {
    // ---- softmax: thread = row of tile t ----------------------------------
    const int t = warp >> 2, rl = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
    const uint32_t ts = tmem_s + t * 2 * kHalf + lanes, to = tmem_o + t * D + lanes;
    const float c = a.scale_log2;
    int64_t unit = u0;
    int it = 0;
    bool dead = false;
    while (unit < u1) {
      const Piece pc = piece_at(p, unit, u1);
      const int r = pc.pair * MR + t * kTileRows + rl;
      const int tok = token_of(p, r), g = r - tok * a.group;
      const bool in = tok < a.T;
      if (!dead) {
        // This warp's 32 rows of Q, a row of 16-byte chunks by D / 8 lanes.
        constexpr int CPR = D / 8, RPP = 32 / CPR;
        const int c = lane % CPR;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)pc.h * a.group * a.q_hs + c * 8;
        uint4 v[32 / RPP];
#pragma unroll
        for (int i = 0; i < 32 / RPP; ++i) {
          const int rr = pc.pair * MR + t * kTileRows + (warp & 3) * 32 + i * RPP + lane / CPR;
          const int tk = token_of(p, rr);
          v[i] = make_uint4(0, 0, 0, 0);
          if (tk < a.T && c * 8 < a.dim) v[i] = *reinterpret_cast<const uint4*>(q + (int64_t)tk * a.q_ts + (int64_t)(rr - tk * a.group) * a.q_hs);
        }
#pragma unroll
        for (int i = 0; i < 32 / RPP; ++i) {
          const int row = (warp & 3) * 32 + i * RPP + lane / CPR;
          *reinterpret_cast<uint4*>(qbuf + t * C::kTileBytes + (c >> 3) * C::kPanelBytes + row * 128 +
                                    (((c & 7) ^ (row & 7)) << 4)) = v[i];
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full[t]);
      }
      float m = WR_NEG_INF, l = 0.f;
      for (int i = 0; i < 2 * pc.n && !dead; ++i, ++it) {  // it: half tiles of this CTA
        const int b = it & 1;
        const uint32_t sb = ts + b * kHalf;
        if (!wait_warp(&s_full[t][b], (it >> 1) & 1)) {
          *abort = 1;
          dead = true;
          break;
        }
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld32(sb, s[0]);
        tmem_ld32(sb + 32, s[1]);
        tmem_wait_lds();
        reg_dep32(s[0]);
        reg_dep32(s[1]);
        const int slot = (it >> 1) % kMaskRing;
        if (s_special[slot]) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t w = s_mask[slot][2 * b + k];
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!((w >> j) & 1)) s[k][j] = 0xff800000u;
          }
        }
        float mx[4] = {WR_NEG_INF, WR_NEG_INF, WR_NEG_INF, WR_NEG_INF};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          mx[j & 2] = fmaxf(mx[j & 2], fmaxf(__uint_as_float(s[0][j]), __uint_as_float(s[0][j + 1])));
          mx[1 + (j & 2)] = fmaxf(mx[1 + (j & 2)], fmaxf(__uint_as_float(s[1][j]), __uint_as_float(s[1][j + 1])));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        if (i == 0) {
          m = top;
        } else {
          const bool up = top > m + kRescale;
          if (__any_sync(0xffffffffu, up)) {
            // O stands still once the last PV issued has ended.
            if (!wait_warp(&pv_done[t][b ^ 1], ((it - 1) >> 1) & 1)) {
              *abort = 1;
              dead = true;
              break;
            }
            tc_fence_after();
            const float nm = up ? top : m;
            const float f = up ? ex2p(m - nm) : 1.f;
            m = nm;
            l *= f;
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              uint32_t o[16];
              tmem_ld16(to + k * 16, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(to + k * 16, o);
            }
          }
        }
        const float base = m == WR_NEG_INF ? 0.f : m;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        // The tiles' exponentials take turns: side by side both tiles wait for
        // the SFUs, then both for the rest, and the SFUs for them.
        if (NT == 2 && (t == 1 || it > 0) && !wait_warp(&turn[t], (t == 1 ? it : it - 1) & 1)) {
          *abort = 1;
          dead = true;
          break;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float x = ex2p(fmaf(__uint_as_float(s[k][2 * j]), c, -base));
            const float y = ex2p(fmaf(__uint_as_float(s[k][2 * j + 1]), c, -base));
            ls[j & 3] += x + y;
            __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
            w[j] = *reinterpret_cast<uint32_t*>(&v);
          }
          tmem_st16(sb + k * 16, w);  // over the scores, all of which are in registers
          if (NT == 2 && k == 0 && lane == 0) mbar_arrive(&turn[t ^ 1]);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[t][b]);
      }
      if (!dead && !wait_warp(&pv_done[t][(it - 1) & 1], ((it - 1) >> 1) & 1)) {
        *abort = 1;
        dead = true;
      }
      // The piece's result.
      const bool whole = pc.u == 0 && pc.n == p.us;
      const int64_t orow = (int64_t)tok * a.hq + pc.h * a.group + g;
      const int64_t prow = ((int64_t)blockIdx.x * 2 + (pc.u == 0 ? 1 : 0)) * MR + t * kTileRows + rl;
      if (!dead) {
        // Sums of 64 columns at a time (32 where D is 64) go through the place
        // of this warp's own 32 rows of Q, whose last product has ended (and
        // which no other warp writes its next rows to), to whole rows: a
        // thread's own row would be 16 bytes here and there.
        tc_fence_after();
        __syncwarp();
        uint8_t* stage = qbuf + t * C::kTileBytes + (warp & 3) * 32 * 128;
        // 32 rows of kCols sums: all in this panel, or 16 in each of two.
        auto place = [](int rw) { return D == 64 ? rw * 128 : (rw >> 4) * C::kPanelBytes + (rw & 15) * 256; };
        constexpr int kCols = D == 64 ? 32 : 64, CH = kCols / 4;  // chunks of 16 bytes a row
#pragma unroll 1
        for (int k = 0; k < D / kCols; ++k) {
#pragma unroll
          for (int j = 0; j < kCols / 16; ++j) {
            uint32_t o[16];
            tmem_ld16(to + k * kCols + j * 16, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + place(lane) + (((j * 4 + e) ^ (lane & 7)) << 4)) =
                  make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          __syncwarp();
          const int c = lane % CH;
#pragma unroll 4
          for (int i = 0; i < 32; i += 32 / CH) {
            const int rw = i + lane / CH;  // row of this warp
            const int rr = pc.pair * MR + t * kTileRows + (warp & 3) * 32 + rw;
            const int tk = token_of(p, rr);
            if (tk < a.T && k * kCols + c * 4 < a.dim) {
              float* op = whole ? a.home + ((int64_t)tk * a.hq + pc.h * a.group + (rr - tk * a.group)) * a.dim
                                : a.part.piece + (prow - lane + rw) * a.dim;
              *reinterpret_cast<uint4*>(op + k * kCols + c * 4) =
                  *reinterpret_cast<const uint4*>(stage + place(rw) + ((c ^ (rw & 7)) << 4));
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      } else {
        l = __int_as_float(0x7fc00000);
        m = 0.f;
      }
      if (in) (whole ? a.home_ml + orow : a.part.piece_ml + prow)[0] = make_float2(m, l);
      unit += pc.n;  // once dead, the pieces that are left get NaN too
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NT * 4 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  griddep_wait();  // this launch counts as complete only after the one before it
}

template <int D, int NT>
cudaError_t launch_tiles(const CUtensorMap& km, const CUtensorMap& vm, const PrefixArgs& p, int grid,
                         cudaStream_t stream) {
  using C = Cfg<D, NT>;
  const void* k = reinterpret_cast<const void*>(k_attn_prefix<D, NT>);
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  void* args[3] = {const_cast<CUtensorMap*>(&km), const_cast<CUtensorMap*>(&vm), const_cast<PrefixArgs*>(&p)};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, k, args);
}

}  // namespace

// Heads of 64, or of up to 128 columns, of which those behind the head arrive
// as zeros.  TMA copies want pages that cut a tile of 128 keys evenly (or the reverse),
// 16 keys at least so that a warp's 32 lanes issue a tile's copies at once,
// and strides other than 0.
bool prefix_tiles_ok(const AttnProblem& p) {
  const PagedKv& c = p.c;
  const bool strides = (c.num_pages == 1 || c.page_stride > 0) && (c.hkv == 1 || c.head_stride > 0) &&
                       (c.page_size == 1 || c.slot_stride > 0);
  const int64_t most = (int64_t)1 << 38;  // elements; tensor maps hold strides below 2^40 bytes
  return c.dtype == WR_DTYPE_BF16 && c.dim >= 64 && c.dim <= 128 && p.scale > 1e-30f && p.scale < 1e30f && c.page_size >= 16 &&
         (c.page_size & (c.page_size - 1)) == 0 && strides && c.page_stride < most && c.head_stride < most &&
         c.slot_stride < most && (int64_t)p.T * (p.hq / c.hkv) * (p.hq / c.hkv) < (int64_t)1 << 31;
}

wr_status_t launch_attn_prefix(const AttnProblem& p, const AttnArgs& a, int row_tile, int grid,
                               cudaStream_t stream) {
  const PagedKv& c = p.c;
  CUtensorMap km, vm;
  const int box_keys = c.page_size < kTileKeys ? c.page_size : kTileKeys;
  const cuuint64_t dims[4] = {(cuuint64_t)c.dim, (cuuint64_t)c.page_size, (cuuint64_t)c.hkv, (cuuint64_t)c.num_pages};
  auto bytes = [&](int64_t stride, int n) { return (cuuint64_t)(n > 1 ? stride * 2 : c.dim * 2); };
  const cuuint64_t strides[3] = {bytes(c.slot_stride, c.page_size), bytes(c.head_stride, c.hkv),
                                 bytes(c.page_stride, c.num_pages)};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_keys, 1, 1};
  wr_status_t st = encode_map(&km, c.k, 4, dims, strides, box);
  if (st == WR_OK) st = encode_map(&vm, c.v, 4, dims, strides, box);
  if (st != WR_OK) return st;
  PrefixArgs x{};
  x.a = a;
  x.pairs = (int)(((int64_t)a.T * a.group + row_tile - 1) / row_tile);
  x.us = (a.prefix + kTileKeys - 1) / kTileKeys;
  x.sp.units = (int64_t)a.hkv * x.pairs * x.us;
  x.sp.ranges = grid < x.sp.units ? grid : x.sp.units;
  x.box = box_keys;
  x.group_inv = a.group == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + a.group - 1) / a.group);
  cudaError_t e;
  const int g = (int)x.sp.ranges;
  if (c.dim == 64)
    e = row_tile == 128 ? launch_tiles<64, 1>(km, vm, x, g, stream) : launch_tiles<64, 2>(km, vm, x, g, stream);
  else
    e = row_tile == 128 ? launch_tiles<128, 1>(km, vm, x, g, stream) : launch_tiles<128, 2>(km, vm, x, g, stream);
  return e == cudaSuccess ? WR_OK : cuda_fail(e, "shared_prefix_attention (prefix tiles) launch");
}

}  // namespace wr
