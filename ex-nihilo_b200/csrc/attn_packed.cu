// attn_packed.cu -- causal attention of packed sequences of different lengths
// with grouped key/value heads, head dim 128, on the 5th-generation tensor
// cores (no counterpart in the reference, which encodes one prompt a call,
// src/encoder.lisp:143-183).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   j <= i + nk - nq,
//
// i over a sequence's nq query rows and j over its nk key rows (the queries
// are its last nq positions); a row that sees no key is 0.  The softmax runs
// in one pass over the keys: with m the running maximum and l the running sum
// of 2^(s - m), a larger m scales l and o by 2^(m_old - m_new).
//
// One CTA = one key/value head of one sequence and two tiles (a, b) of
// queries that share every K/V tile.  A tile's 128 rows are 128 / g tokens
// times the g query heads that read this key/value head, so K and V are
// loaded once a group, not once a query head, and a short prompt still fills
// its tiles (a 24-token prompt with g = 4: 96 rows, not 24).  Keys are taken
// 64 at a time ("units"; loads are 128 keys, two units), each tile only as
// far as its last row sees.  Roles, as in the single-sequence kernel of
// attention.cu:
//   warp 0      TMA: Q_a, Q_b once; K_t, V_t through a ring of 4 slots
//   warp 1, 2   tcgen05.mma of tile a, b: S_x(u) = Q_x K(u)^T into one of two
//               TMEM buffers, O_x += P_x(u) V(u) with P_x read from TMEM
//   warps 3..10 softmax of tile a, then b: one row a thread; P_x(u) written
//               over S_x(u); O_x rescaled in TMEM only when the row maximum
//               grows by more than 2^8 (P then stays below 2^8, in range of
//               both 16-bit types)
// The sums and maxima are fp32; P is rounded to the inputs' 16-bit type (the
// tensor core's operand), o once at the end.
//
// A hidden key's P is 0, and 0 times a V that is infinite or NaN would still
// be NaN in the tensor core: such V rows can belong to the next sequence or to
// a later token.  So an output row that comes out not finite is looked at
// again (mend_row): when a hidden V row of its last units is not finite, the
// row is computed anew over its visible keys alone.
#include "exn_device.cuh"
#include "exn_internal.h"

namespace exn {

int make_tmap(CUtensorMap* m, CUtensorMapDataType type, const void* base, int rank, const uint64_t* dims,
              const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle);

namespace {

constexpr int PK_THREADS = 352;
constexpr int TILE = 128;             // rows per query tile, keys per K/V load
constexpr int UNIT = 64;              // keys per S tile
constexpr int HALF = TILE * 128;      // bytes of one 64-column swizzled half of a 128 x 128 16-bit tile
constexpr int TILE_BYTES = 2 * HALF;  // 32 KB
constexpr int SLOTS = 4;              // K_0 V_0 K_1 V_1 ... stream through 4 slots
constexpr int OFF_QA = 0, OFF_QB = TILE_BYTES, OFF_SLOT = 2 * TILE_BYTES, OFF_BAR = (2 + SLOTS) * TILE_BYTES;
constexpr int PK_SMEM = OFF_BAR + 256 + 1024;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

// kind::f16 instruction descriptor for 16-bit operands of one type (bf16 or fp16) and fp32 sums
template <bool F16>
constexpr uint32_t idesc16(int m, int n, bool b_mn) {
  return F16 ? (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
                   (static_cast<uint32_t>(m >> 4) << 24)
             : idesc_bf16(m, n, false, b_mn);
}

struct Bars {
  uint64_t q_full, slot_full[SLOTS], slot_empty[SLOTS];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][S buffer]
  uint64_t pv_done[2], o_full[2], done[2];
  uint32_t tmem_slot;
  int abort_flag;
  int seq;  // the item's sequence, -1: none
};

template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (F16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  return pack_bf16x2(lo, hi);
}

// One output row by one warp (lane l: dims 4l .. 4l+3), for a row that came out not finite.  Keys
// 0 .. LIM are visible; rows LIM+1 .. LAST of V were multiplied by P = 0 as well.  When one of
// those is not finite the row is computed over its visible keys, with fp32 P; else it stays (what
// it sees is not finite itself).
template <bool F16>
__device__ __noinline__ void mend_row(const uint16_t* q, const uint16_t* k, long long ld_k, const uint16_t* v,
                                      long long ld_v, int lim, int last, float scale_log2, uint16_t* out) {
  const int d = (threadIdx.x & 31) * 4;
  bool hidden_bad = false;
  for (int j = max(lim + 1, 0); j <= last; ++j) {
    const uint2 w = *reinterpret_cast<const uint2*>(v + j * ld_v + d);
    const float2 a = unpack16<F16>(w.x), b = unpack16<F16>(w.y);
    hidden_bad |= !(isfinite(a.x) && isfinite(a.y) && isfinite(b.x) && isfinite(b.y));
  }
  if (!__any_sync(0xffffffffu, hidden_bad)) return;
  const uint2 qw = *reinterpret_cast<const uint2*>(q + d);
  const float2 q0 = unpack16<F16>(qw.x), q1 = unpack16<F16>(qw.y);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j <= lim; ++j) {  // none for a row that sees no key
    const uint2 kw = *reinterpret_cast<const uint2*>(k + j * ld_k + d);
    const uint2 vw = *reinterpret_cast<const uint2*>(v + j * ld_v + d);
    const float2 k0 = unpack16<F16>(kw.x), k1 = unpack16<F16>(kw.y);
    float s = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= scale_log2;
    if (s > m) {
      const float c = exp2f(m - s);
      l *= c;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= c;
      m = s;
    }
    const float p = m == -INFINITY && !(s != s) ? 0.f : exp2f(s - m);
    l += p;
    const float2 v0 = unpack16<F16>(vw.x), v1 = unpack16<F16>(vw.y);
    o[0] += p * v0.x;
    o[1] += p * v0.y;
    o[2] += p * v1.x;
    o[3] += p * v1.y;
    // nothing changes any more once the whole row is NaN
    if ((j & 63) == 63 &&
        __all_sync(0xffffffffu, o[0] != o[0] && o[1] != o[1] && o[2] != o[2] && o[3] != o[3])) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(out + d) =
      make_uint2(pack16<F16>(o[0] * inv, o[1] * inv), pack16<F16>(o[2] * inv, o[3] * inv));
}

template <bool F16>
__global__ void __launch_bounds__(PK_THREADS, 1)
    k_packed(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
             const __grid_constant__ CUtensorMap tmV, const PackedArgs p, int tpt, int nslots, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + OFF_BAR);
  volatile int* abort_flag = &bars->abort_flag;
  constexpr uint32_t IDESC_S = idesc16<F16>(128, UNIT, false);
  constexpr uint32_t IDESC_PV = idesc16<F16>(128, 128, true);  // V is MN-major (dims contiguous)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = p.heads / p.kv_heads;
  const int kvh = blockIdx.x % p.kv_heads;
  // Work item: a pair of tiles.  Sequence s owns the pair slots from floor(start_s / (2 tpt)) + s
  // on; the distance to the next sequence's first slot is at least ceil(length / (2 tpt)), so the
  // host knows the count of slots without the lengths.  Later slots first: a sequence's last
  // tiles see the most keys.
  const int slot = nslots - 1 - static_cast<int>(blockIdx.x) / p.kv_heads;
  if (threadIdx.x == 0) bars->seq = -1;
  griddep_wait();  // the offsets may be the previous kernel's output, as Q, K and V
  griddep_launch();
  __syncthreads();
  for (int s = threadIdx.x; s < p.nseq; s += PK_THREADS) {
    const long long a = p.q_offsets[s], b = p.q_offsets[s + 1];
    if (a < 0 || b < a || b > p.rows) {
      if (blockIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      continue;
    }
    const long long first = a / (2 * tpt) + s;
    if (slot >= first && slot < first + (b - a + 2 * tpt - 1) / (2 * tpt)) bars->seq = s;
  }
  __syncthreads();
  const int seq = bars->seq;
  if (seq < 0) return;
  const int q_start = p.q_offsets[seq], nq = p.q_offsets[seq + 1] - q_start;
  long long k_start;
  int nk;
  if (p.kv_lens) {
    k_start = p.kv_stride * seq;
    nk = p.kv_lens[seq];
  } else {
    k_start = p.kv_offsets[seq];
    nk = p.kv_offsets[seq + 1] - static_cast<int>(k_start);
  }
  if (k_start < 0 || nk < 0 || k_start + nk > p.kv_rows) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    return;
  }
  const int t0 = (slot - (q_start / (2 * tpt) + seq)) * 2 * tpt;  // the pair's first token within the sequence
  const int tiles = nq - t0 > tpt ? 2 : 1;
  const int delta = nk - nq;  // token t sees keys 0 .. t + delta
  int nu[2] = {0, 0};         // units each tile's last row sees
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (x < tiles) {
      const int seen = min(nq, t0 + (x + 1) * tpt) + delta;
      nu[x] = seen > 0 ? (seen + UNIT - 1) / UNIT : 0;
    }
  const int nunits = max(nu[0], nu[1]);
  const int nloads = (nunits + 1) / 2;
  uint16_t* const out = static_cast<uint16_t*>(p.out);

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], tiles);
    }
    for (int x = 0; x < 2; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[x][b], 1);
        mbar_init(&bars->p_full[x][b], 4);
      }
      mbar_init(&bars->pv_done[x], 1);
      mbar_init(&bars->o_full[x], 1);
      mbar_init(&bars->done[x], 1);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_slot;
  // TMEM columns: S_a buffers [0,64) [64,128), S_b [128,192) [192,256), O_a [256,384), O_b [384,512)

  if (warp == 0) {
    if (lane == 0 && nunits > 0) {
      tma_prefetch(&tmQ);
      tma_prefetch(&tmK);
      tma_prefetch(&tmV);
      // a tile of Q: the box (64 dims, g heads, tpt tokens), rows token-major; rows of the tile
      // past g tpt stay as they are and are never stored
      mbar_arrive_expect_tx(&bars->q_full, tiles * 2 * g * tpt * 128);
      for (int x = 0; x < tiles; ++x)
        for (int hf = 0; hf < 2; ++hf)
          tma_load_3d(smem + (x ? OFF_QB : OFF_QA) + hf * HALF, &tmQ, &bars->q_full, hf * 64, kvh * g,
                      q_start + t0 + x * tpt);
      int issued = 0;
      for (int t = 0; t < 2 * nloads; ++t) {
        const int sl = t % SLOTS;
        const uint32_t use = static_cast<uint32_t>(t / SLOTS);
        if (!mbar_wait(&bars->slot_empty[sl], (use & 1) ^ 1, abort_flag, status, STATUS_TIMEOUT_ATTN)) break;
        mbar_arrive_expect_tx(&bars->slot_full[sl], TILE_BYTES);
        const CUtensorMap* map = (t & 1) ? &tmV : &tmK;
        for (int hf = 0; hf < 2; ++hf)
          tma_load_2d(smem + OFF_SLOT + sl * TILE_BYTES + hf * HALF, map, &bars->slot_full[sl], kvh * 128 + hf * 64,
                      static_cast<int>(k_start) + (t >> 1) * TILE);
        issued = t + 1;
      }
      if (*abort_flag) {  // the copies in flight land before the CTA leaves
        volatile int no_abort = 0;
        mbar_wait(&bars->q_full, 0, &no_abort, nullptr, 0);
        for (int t = issued - SLOTS < 0 ? 0 : issued - SLOTS; t < issued; ++t)
          mbar_wait(&bars->slot_full[t % SLOTS], static_cast<uint32_t>(t / SLOTS) & 1, &no_abort, nullptr, 0);
      }
    }
  } else if (warp <= 2) {
    if (lane == 0 && warp - 1 < tiles && nunits > 0) {
      // ---- the MMAs of tile x (descriptors as 32-bit low words over a common high word)
      const int x = warp - 1;
      const int n = nu[x];
      const uint32_t dhi = static_cast<uint32_t>(sdesc_sw128(0, 16, 1024) >> 32);
      const uint32_t qlo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + (x ? OFF_QB : OFF_QA)), 16, 1024));
      const uint32_t klo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + OFF_SLOT), 16, 1024));    // K-major
      const uint32_t vlo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + OFF_SLOT), HALF, 1024));  // MN-major
      const uint32_t s_tm = tmem + x * 128, o_tm = tmem + 256 + x * 128;
      auto issue_s = [&](int u) {
        const uint32_t k = klo + ((((u >> 1) * 2) % SLOTS) * TILE_BYTES + (u & 1) * UNIT * 128) / 16;
        const uint32_t d = s_tm + (u & 1) * UNIT;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t o = ((kk >> 2) * HALF + (kk & 3) * 32) / 16;
          umma_ss_lo(d, qlo + o, k + o, dhi, IDESC_S, kk ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int u) {
        const uint32_t v = vlo + ((((u >> 1) * 2 + 1) % SLOTS) * TILE_BYTES + (u & 1) * UNIT * 128) / 16;
        const uint32_t a = s_tm + (u & 1) * UNIT;
#pragma unroll
        for (int kk = 0; kk < UNIT / 16; ++kk)
          umma_ts_lo(o_tm, a + kk * 8, v + kk * 2048 / 16, dhi, IDESC_PV, (u > 0 || kk) ? 1u : 0u);
      };
      auto wait_load = [&](int t) {
        return mbar_wait(&bars->slot_full[t % SLOTS], static_cast<uint32_t>(t / SLOTS) & 1, abort_flag, status,
                         STATUS_TIMEOUT_ATTN);
      };
      bool ok = mbar_wait(&bars->q_full, 0, abort_flag, status, STATUS_TIMEOUT_ATTN);
      if (ok && n > 0 && (ok = wait_load(0))) {
        tc_fence_after();
        for (int u = 0; u < 2 && u < n; ++u) {
          issue_s(u);
          umma_commit(&bars->s_full[x][u]);
        }
        umma_commit(&bars->slot_empty[0]);  // K_0: both its units issued
      }
      for (int u = 0; u < n && ok; ++u) {
        const int b = u & 1;
        const bool more = u + 2 < n;
        if (b == 0 && !(ok = wait_load(2 * (u >> 1) + 1))) break;  // V(u)
        if (!(ok = mbar_wait(&bars->p_full[x][b], static_cast<uint32_t>(u >> 1) & 1, abort_flag, status,
                             STATUS_TIMEOUT_ATTN)))
          break;
        tc_fence_after();
        issue_pv(u);
        umma_commit(&bars->pv_done[x]);
        if (u + 1 == n) umma_commit(&bars->o_full[x]);
        if (more) {
          if (b == 0 && !(ok = wait_load(2 * ((u + 2) >> 1)))) break;  // K(u + 2)
          issue_s(u + 2);
          umma_commit(&bars->s_full[x][b]);
        }
        // this tile's share of freeing the slots whose last reader was just issued
        if (b == 1 || u + 1 == n) umma_commit(&bars->slot_empty[(2 * (u >> 1) + 1) % SLOTS]);   // V(u)
        if (more && (b == 1 || u + 3 == n)) umma_commit(&bars->slot_empty[(2 * ((u + 2) >> 1)) % SLOTS]);
      }
      // the loads only the other tile reads: this tile's share once each has landed
      for (int t = 2 * ((n + 1) / 2); t < 2 * nloads && ok; ++t) {
        if (!(ok = wait_load(t))) break;
        umma_commit(&bars->slot_empty[t % SLOTS]);
      }
      umma_commit(&bars->done[x]);  // every MMA queued above has finished before TMEM is released
      volatile int no_abort = 0;
      mbar_wait(&bars->done[x], 0, &no_abort, nullptr, 0);
    }
  } else if ((warp - 3) >> 2 < tiles) {
    // ---- softmax: tile x, TMEM lane quarter wq, row r of the tile
    const int x = (warp - 3) >> 2;
    const int n = nu[x];
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const int tok = r / g;
    const int t = t0 + x * tpt + tok;  // token within the sequence
    const bool live = tok < tpt && t < nq;
    const int lim = live ? t + delta : n * UNIT;  // last visible key (< 0: none)
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + x * 128;
    const uint32_t o_addr = tmem + lane_off + 256 + x * 128;
    float m = -INFINITY, lsum = 0.f;
    bool ok = true;
    const uint64_t sc2 = f2(p.scale_log2, p.scale_log2);
    // the two tiles' exponentials take turns on each scheduler (attention.cu); tile a's turns end
    // with its last unit, which is never after tile b's
    const uint32_t my_turn = (x ? 5u : 1u) + static_cast<uint32_t>(wq);
    const uint32_t other_turn = (x ? 1u : 5u) + static_cast<uint32_t>(wq);
    const int turns = tiles == 2 ? nu[0] : 0;
    if (turns > 0 && x == 1) asm volatile("bar.arrive %0, 64;" ::"r"(other_turn) : "memory");  // tile a goes first
    for (int u = 0; u < n; ++u) {
      const int b = u & 1;
      ok = ok && mbar_wait_uniform(&bars->s_full[x][b], static_cast<uint32_t>(u >> 1) & 1, abort_flag, status,
                                   STATUS_TIMEOUT_ATTN);
      float s[UNIT];
      float nm = 0.f;
      if (ok) {
        tc_fence_after();
        {
          uint32_t rr[UNIT];
          tmem_ld64_conv(s_addr + b * UNIT, rr);
#pragma unroll
          for (int i = 0; i < UNIT; ++i) s[i] = __uint_as_float(rr[i]);
        }
        const int key0 = u * UNIT;
        if (__any_sync(0xffffffffu, key0 + UNIT - 1 > lim)) {
#pragma unroll
          for (int c = 0; c < UNIT; ++c)
            if (key0 + c > lim) s[c] = -INFINITY;
        }
        float m8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmax3(s[i], s[8 + i], s[16 + i]);
#pragma unroll
        for (int c = 24; c < UNIT - 8; c += 16)
#pragma unroll
          for (int i = 0; i < 8; ++i) m8[i] = fmax3(m8[i], s[c + i], s[c + 8 + i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(m8[i], s[UNIT - 8 + i]);
        const float mx = fmaxf(fmax3(m8[0], m8[1], m8[2]), fmax3(fmax3(m8[3], m8[4], m8[5]), m8[6], m8[7]));
        const float m_new = fmaxf(m, mx * p.scale_log2);
        const bool need = m_new > m + RESCALE_THRESHOLD;
        const float alpha = need ? fast_exp2(m - m_new) : 1.f;
        lsum *= alpha;
        m = need ? m_new : m;
        nm = m == -INFINITY ? 0.f : -m;  // nothing seen yet: every P is 2^-inf = 0
        if (u > 0 && __any_sync(0xffffffffu, need)) {
          ok = mbar_wait_uniform(&bars->pv_done[x], static_cast<uint32_t>(u - 1) & 1, abort_flag, status,
                                 STATUS_TIMEOUT_ATTN);
          if (ok) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t ov[32];
              tmem_ld32(o_addr + c * 32, ov);
#pragma unroll
              for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
              tmem_st32(o_addr + c * 32, ov);
            }
            tmem_st_wait();
          }
        }
      }
      if (u < turns) asm volatile("bar.sync %0, 64;" ::"r"(my_turn) : "memory");
      uint32_t pk[UNIT / 2];  // P as 16-bit pairs: key 2c and 2c+1 in column c
      if (ok) {
        const uint64_t nm2 = f2(nm, nm);
        uint64_t ps2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c8 = 0; c8 < UNIT / 8; ++c8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x0, x1;
            f2_split(ffma2(f2(s[c8 * 8 + 2 * i], s[c8 * 8 + 2 * i + 1]), sc2, nm2), x0, x1);
            const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
            ps2[i] = fadd2(ps2[i], f2(e0, e1));
            pk[c8 * 4 + i] = pack16<F16>(e0, e1);
          }
        }
        float a0, a1;
        f2_split(fadd2(fadd2(ps2[0], ps2[1]), fadd2(ps2[2], ps2[3])), a0, a1);
        lsum += a0 + a1;
      }
      if (u < turns && (x == 0 || u + 1 < turns)) asm volatile("bar.arrive %0, 64;" ::"r"(other_turn) : "memory");
      if (ok) {
        tmem_st32_conv(s_addr + b * UNIT, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[x][b]);
      }
    }
    const int head = kvh * g + r - tok * g;
    uint16_t* dst = out + static_cast<long long>(q_start + t) * p.ld_out + head * 128;
    if (n > 0) {
      if (ok && mbar_wait_uniform(&bars->o_full[x], 0, abort_flag, status, STATUS_TIMEOUT_ATTN)) {
        tc_fence_after();
        const bool none = lsum == 0.f;
        const float inv = none ? 0.f : 1.f / lsum;
        float finite = 0.f;  // 0 times every output: NaN when one is not finite
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t rr[32];
          tmem_ld32(o_addr + c * 32, rr);
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            o[i] = __uint_as_float(rr[i]) * inv;
            finite = fmaf(o[i], 0.f, finite);
          }
          if (live) {
            uint4* d4 = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              d4[i] = make_uint4(pack16<F16>(o[8 * i], o[8 * i + 1]), pack16<F16>(o[8 * i + 2], o[8 * i + 3]),
                                 pack16<F16>(o[8 * i + 4], o[8 * i + 5]), pack16<F16>(o[8 * i + 6], o[8 * i + 7]));
          }
        }
        __syncwarp();
        unsigned bad = __ballot_sync(0xffffffffu, live && finite != 0.f);
        while (bad) {
          const int src = __ffs(bad) - 1;
          bad &= bad - 1;
          const int rt = __shfl_sync(0xffffffffu, t, src), rh = __shfl_sync(0xffffffffu, head, src);
          const int rl = __shfl_sync(0xffffffffu, lim, src);
          const long long rows_end = p.kv_rows - k_start;  // rows past the tensor were read as zeros
          const int last = static_cast<int>(min(static_cast<long long>(n) * UNIT, rows_end)) - 1;
          const uint16_t* kb = static_cast<const uint16_t*>(p.k) + k_start * p.ld_k + kvh * 128;
          const uint16_t* vb = static_cast<const uint16_t*>(p.v) + k_start * p.ld_v + kvh * 128;
          mend_row<F16>(static_cast<const uint16_t*>(p.q) + static_cast<long long>(q_start + rt) * p.ld_q + rh * 128,
                        kb, p.ld_k, vb, p.ld_v, rl, last, p.scale_log2,
                        out + static_cast<long long>(q_start + rt) * p.ld_out + rh * 128);
          __syncwarp();
        }
      }
    } else if (live) {  // no row of the tile sees a key
      uint4* d4 = reinterpret_cast<uint4*>(dst);
#pragma unroll
      for (int i = 0; i < 16; ++i) d4[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

int packed_prepare() {
  cudaError_t e = cudaFuncSetAttribute(k_packed<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PK_SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_packed<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PK_SMEM);
  return static_cast<int>(e);
}

int packed_launch(const PackedArgs& a, int* d_status, cudaStream_t st) {
  const int g = a.heads / a.kv_heads;
  const int tpt = TILE / g;  // tokens a tile
  const CUtensorMapDataType type = a.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tk, tv;
  const uint64_t dq[3] = {128, static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.rows)};
  const uint64_t sq[2] = {256, static_cast<uint64_t>(a.ld_q) * 2};
  const uint32_t bq[3] = {64, static_cast<uint32_t>(g), static_cast<uint32_t>(tpt)};
  const uint64_t dk[2] = {static_cast<uint64_t>(a.kv_heads) * 128,
                          static_cast<uint64_t>(a.kv_rows > 0 ? a.kv_rows : 1)};  // no key row: no load either
  const uint64_t sk[1] = {static_cast<uint64_t>(a.ld_k) * 2}, sv[1] = {static_cast<uint64_t>(a.ld_v) * 2};
  const uint32_t bk[2] = {64, TILE};
  if (make_tmap(&tq, type, a.q, 3, dq, sq, bq, CU_TENSOR_MAP_SWIZZLE_128B) ||
      make_tmap(&tk, type, a.k, 2, dk, sk, bk, CU_TENSOR_MAP_SWIZZLE_128B) ||
      make_tmap(&tv, type, a.v, 2, dk, sv, bk, CU_TENSOR_MAP_SWIZZLE_128B))
    return -4;
  const long long nslots = a.rows / (2 * tpt) + a.nseq;
  if (nslots * a.kv_heads > 0x7fffffffll) return -1;
  return static_cast<int>(launch_pdl(a.f16 ? k_packed<true> : k_packed<false>,
                                     dim3(static_cast<unsigned>(nslots * a.kv_heads)), dim3(PK_THREADS), PK_SMEM, st, tq,
                                     tk, tv, a, tpt, static_cast<int>(nslots), d_status));
}

}  // namespace exn
