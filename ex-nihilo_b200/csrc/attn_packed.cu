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
// A work item is one key/value head of one sequence and two tiles (a, b) of queries that share every K/V
// tile.  A tile's 128 rows are 128 / g tokens times the g query heads that read this key/value head, so K
// and V are loaded once a group, not once a query head, and a short prompt still fills its tiles (a
// 24-token prompt with g = 4: 96 rows, not 24).  Keys are taken 64 at a time ("units"; loads are 128 keys,
// two units), each tile only as far as its last row sees.
//
// One CTA an SM takes items one after another, the longest first within a sequence: the grid has a CTA an
// item, and a running CTA takes over those that have not started (cluster launch control), so the SMs
// stay evenly loaded without a counter in memory, and barriers, TMEM and tensor maps are set up once.
// SPLIT: where there are too few items of long sequences for the SMs, a cluster of 2, 4 or 8 CTAs shares
// an item, each a part of its keys, and joins the parts through shared memory: with row maxima m_c,
// sums l_c and outputs o_c of the parts and M = max m_c, o = sum 2^(m_c - M) o_c / sum 2^(m_c - M) l_c.
// When there are more items than clusters, the longest ones are shared and a cluster's CTAs take one each
// of the others.
// Roles, as in the single-sequence kernel of attention.cu:
//   warp 0      finds the next item; TMA: Q_a, Q_b once an item; K_t, V_t through a ring of 4 slots, the next
//               item's behind the last one's
//   warp 1, 2   tcgen05.mma of tile a, b: S_x(u) = Q_x K(u)^T into one of two TMEM buffers, O_x += P_x(u) V(u)
//               with P_x read from TMEM; the next item's first S while the last O is stored
//   warps 3..10 softmax of tile a, then b: one row a thread; P_x(u) written over S_x(u); O_x rescaled in TMEM
//               only when the row maximum grows by more than 2^8 (P then stays below 2^8, in range of
//               both 16-bit types)
// The sums and maxima are fp32; P is rounded to the inputs' 16-bit type, since the
// tensor core multiplies operands of one type, and o once at the end.  Against 64 bits that makes an output's
// relative error 0.0021 in bf16 and 0.00025 in fp16 at 2000 to 8192 keys, where fp32 weights leave the output's own
// rounding, 0.0016 and 0.00020.  In fp16 a weight below 2^-25 of the largest is 0.
//
// Bound by the chain S, maximum, exponentials, P, PV of a unit, 0.98 us for both tiles: at 8192 causal rows of
// 32 heads over 8 (452 to 463 us from box to box, 1190 TFLOP/s) the tensor pipe is busy 55 % of the time, the
// exponentials' 56 %, the schedulers 42 %.  Eleven warps leave a thread 168 registers, of which 8 to 24 bytes
// spill.  A fourth of the exponentials as polynomials (491 us, 465 then), no turns between the two tiles (476) and
// two warps a row (520) were slower.  A short item costs about 5 us besides its units, most of which overlaps
// with the next one's loads; a launch of one prompt of 27 rows takes 6.5 us.
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
constexpr int PK_SMEM = OFF_BAR + 512 + 1024;
constexpr int MIN_SHARED = 768;            // keys of an item that is worth a cluster
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

// kind::f16 instruction descriptor for 16-bit operands of one type (bf16 or fp16) and fp32 sums
template <bool F16>
constexpr uint32_t idesc16(int m, int n, bool b_mn) {
  return F16 ? (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
                   (static_cast<uint32_t>(m >> 4) << 24)
             : idesc_bf16(m, n, false, b_mn);
}

// A work item; n 0 in both tiles: no row of it sees a key
struct Item {
  int q_start, nq, t0, tiles;  // the sequence's first query row and rows, the item's first token and tiles
  int delta, nu[2], nloads;    // token t sees keys 0 .. t + delta; units of each tile; 128-key loads
  int kvh;                     // key/value head; -1: no more items
  int key0, share;             // the CTA's first key; whether the cluster's CTAs share the item
  int k_start;                 // the sequence's first key row
};

struct Bars {
  uint64_t q_full[2], q_empty[2], slot_full[SLOTS], slot_empty[SLOTS];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][S buffer]
  uint64_t pv_done[2], o_full[2], done[2];
  uint64_t item_full[2], item_empty[2], claim_full;
  uint4 claim;  // cluster launch control's answer
  Item item[2];
  uint32_t tmem_slot;
  int abort_flag;
};

// Ask for a CTA of the grid that has not started; the answer's 16 bytes land in DST and complete BAR
__device__ __forceinline__ void claim_request(void* dst, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(dst)),
               "r"(smem_u32(bar))
               : "memory");
}
// the CTA's index that the answer gives us, -1: none was left
__device__ __forceinline__ int claim_answer(const void* src) {
  int x, got;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.s32 %1, 1, 0, p;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, r;\n\t}"
      : "=r"(x), "=r"(got)
      : "r"(smem_u32(src))
      : "memory");
  return got ? x : -1;
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

static_assert(sizeof(Bars) <= 512, "the barriers' room");

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

// 32 bytes at a 32-byte boundary
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// the sum of X over the lanes before this one
__device__ __forceinline__ int warp_before(int x) {
  const int lane = threadIdx.x & 31;
  int sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  return sum - x;
}

template <bool F16, bool SPLIT>
__global__ void __launch_bounds__(PK_THREADS, 1)
    k_packed(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
             const __grid_constant__ CUtensorMap tmV, const PackedArgs p, int tpt, int nslots, int fit,
             int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + OFF_BAR);
  volatile int* abort_flag = &bars->abort_flag;
  constexpr uint32_t IDESC_S = idesc16<F16>(128, UNIT, false);
  constexpr uint32_t IDESC_PV = idesc16<F16>(128, 128, true);  // V is MN-major (dims contiguous)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = p.heads / p.kv_heads;
  uint16_t* const out = static_cast<uint16_t*>(p.out);
  const int parts = SPLIT ? static_cast<int>(cluster_nctarank()) : 1, part = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], 2);  // free once both tiles' MMAs are done with it
    }
    for (int x = 0; x < 2; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[x][b], 1);
        mbar_init(&bars->p_full[x][b], 4);
      }
      mbar_init(&bars->q_full[x], 1);
      mbar_init(&bars->q_empty[x], 1);
      mbar_init(&bars->pv_done[x], 1);
      mbar_init(&bars->o_full[x], 1);
      mbar_init(&bars->done[x], 1);
      mbar_init(&bars->item_full[x], 1);
      mbar_init(&bars->item_empty[x], 10);  // the two MMA threads and eight softmax warps
    }
    mbar_init(&bars->claim_full, 1);
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
  griddep_wait();  // the offsets may be the previous kernel's output, as Q, K and V
  griddep_launch();
  if (blockIdx.x == 0)  // what is wrong with the offsets is reported once; the items leave it out
    for (int s = threadIdx.x; s < p.nseq; s += PK_THREADS) {
      const int a = p.q_offsets[s], b = p.q_offsets[s + 1];
      if (a < 0 || b < a || b > p.rows) atomicOr(status, STATUS_BAD_ARG);
    }

  // The waits for the next item are the only ones that do not look at the abort flag, so every role goes through
  // the same items, with the work left out once a wait has run out, and the tiles' warps stay in step.  The
  // producer, whose own waits are shorter, ends the list.
  volatile int no_abort = 0;
  auto wait_item = [&](uint64_t* bar, uint32_t parity, int limits = 16) {  // one thread
    volatile int none = 0;
    return mbar_wait(bar, parity, &none, status, STATUS_TIMEOUT_ATTN, limits * EXN_WAIT_NS);
  };

  bool joined = false;
  if (warp == 0) {
    // ---- the items: pairs of query tiles, times the key/value heads.  A lane has a run of the sequences and knows
    // how many items come before it.  Up to 32 sequences, a lane each, go in the order of their keys, the longest
    // first, and a sequence's last tiles, which see the most, before its first: an item that starts late is then
    // short (1024 rows over 5555 keys, 300 over 300 and 512 over 8192, 32 heads over 8: 160 us so, 200 in their
    // own order).  The host knows a bound of the count without the lengths.
    const int pair = 2 * tpt;
    struct Sequence {
      int q0, q1, k0, nk, pairs;  // rows, keys, items a head
    };
    int decrease = p.nseq;  // the sequences from the first whose offsets decrease on are left out: their rows may be
                            // earlier ones', and there may be more items than the host's bound
    auto read = [&](int s) {
      Sequence x;
      x.q0 = p.q_offsets[s];
      x.q1 = p.q_offsets[s + 1];
      long long start;
      if (p.kv_lens) {
        start = p.kv_stride * s;
        x.nk = p.kv_lens[s];
      } else {
        start = p.kv_offsets[s];
        x.nk = p.kv_offsets[s + 1] - static_cast<int>(start);
      }
      x.pairs = s >= decrease || x.q0 < 0 || x.q1 < x.q0 || x.q1 > p.rows ? 0 : (x.q1 - x.q0 + pair - 1) / pair;
      if (x.pairs && (start < 0 || x.nk < 0 || start + x.nk > p.kv_rows)) {
        atomicOr(status, STATUS_BAD_ARG);
        x.pairs = 0;
      }
      x.k0 = static_cast<int>(start);
      return x;
    };
    const int run = (p.nseq + 31) / 32;
    const bool sorted = run == 1;
    Sequence mine = {0, 0, 0, 0, 0};
    int pairs = 0, first = 0;  // of the lane's run: its items a head, those before it
    if (sorted) {
      if (lane < p.nseq) mine = read(lane);
      const unsigned less = __ballot_sync(0xffffffffu, mine.q1 < mine.q0);
      if (less && lane >= __ffs(less) - 1) mine.pairs = 0;
      pairs = mine.pairs;
      for (int j = 0; j < p.nseq; ++j) {
        const int other = __shfl_sync(0xffffffffu, mine.nk, j), n = __shfl_sync(0xffffffffu, pairs, j);
        if (other > mine.nk || (other == mine.nk && j < lane)) first += n;
      }
    } else {
      int less = p.nseq;
      for (bool again = true; again;) {
        decrease = less;
        pairs = 0;
        for (int s = lane * run; s < min(p.nseq, lane * run + run); ++s) {
          const Sequence x = read(s);
          pairs += x.pairs;
          if (x.q1 < x.q0) less = min(less, s);
        }
        less = __reduce_min_sync(0xffffffffu, less);
        again = less < decrease;  // once more without those behind it
      }
      first = warp_before(pairs);
    }
    auto find = [&](int index, Item& x) -> bool {  // by the whole warp; false: no such item
      int at = index / p.kv_heads - first;
      unsigned owner = __ballot_sync(0xffffffffu, at >= 0 && at < pairs);
      if (!owner) return false;
      int src = __ffs(owner) - 1;
      Sequence mine_now = mine;
      if (!sorted) {  // the owner's run, 32 sequences at a time
        at = __shfl_sync(0xffffffffu, at, src);
        const int end = min(p.nseq, src * run + run);
        for (int s0 = src * run;; s0 += 32) {
          if (s0 >= end) return false;  // not before the offsets change under the kernel
          mine_now = s0 + lane < end ? read(s0 + lane) : Sequence{0, 0, 0, 0, 0};
          const int before = warp_before(mine_now.pairs);
          owner = __ballot_sync(0xffffffffu, at >= before && at < before + mine_now.pairs);
          if (owner) {
            at -= before;
            break;
          }
          at -= __shfl_sync(0xffffffffu, before + mine_now.pairs, 31);
        }
        src = __ffs(owner) - 1;
      }
      const int i = __shfl_sync(0xffffffffu, mine_now.pairs - 1 - at, src), a = __shfl_sync(0xffffffffu, mine_now.q0, src),
                b = __shfl_sync(0xffffffffu, mine_now.q1, src), from = __shfl_sync(0xffffffffu, mine_now.k0, src),
                keys = __shfl_sync(0xffffffffu, mine_now.nk, src);
      x.t0 = i * pair;
      x.q_start = a;
      x.nq = b - a;
      x.k_start = from;
      x.kvh = index % p.kv_heads;
      x.tiles = x.nq - x.t0 > tpt ? 2 : 1;
      x.delta = keys - x.nq;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int seen = i < x.tiles ? min(x.nq, x.t0 + (i + 1) * tpt) + x.delta : 0;
        x.nu[i] = seen > 0 ? (seen + UNIT - 1) / UNIT : 0;
      }
      x.nloads = (max(x.nu[0], x.nu[1]) + 1) / 2;
      x.key0 = 0;
      if (SPLIT && x.share) {  // this CTA's share of the 128-key loads
        const int l0 = x.nloads * part / parts, l1 = x.nloads * (part + 1) / parts;
        x.key0 = l0 * TILE;
        x.nloads = l1 - l0;
#pragma unroll
        for (int i = 0; i < 2; ++i) x.nu[i] = min(max(x.nu[i] - 2 * l0, 0), 2 * (l1 - l0));
      }
      return true;
    };
    // The next item is asked for late, near the end of the item at hand: it may be one that would soon have found
    // an SM of its own.
    uint32_t claims = 0;
    bool ok = true, asked = false, ended = SPLIT;
    auto ask = [&] {
      if (lane == 0) claim_request(&bars->claim, &bars->claim_full);
      asked = true;
    };
    auto next_item = [&](Item& x) {  // kvh -1: no more
      x.kvh = -1;
      while (!ended && ok) {
        if (!asked) ask();
        if (!__shfl_sync(0xffffffffu, lane == 0 ? wait_item(&bars->claim_full, claims & 1, 1) : true, 0)) {
          ok = false;
          return;
        }
        ++claims;
        asked = false;
        const int index = claim_answer(&bars->claim);
        ended = index < 0;
        fence_proxy_async_smem();  // the answer is read before the next one is written
        __syncwarp();
        if (!ended && find(index, x)) return;
        x.kvh = -1;
      }
    };
    if (lane == 0) {
      tma_prefetch(&tmQ);
      tma_prefetch(&tmK);
      tma_prefetch(&tmV);
    }
    Item cur;
    int index = static_cast<int>(blockIdx.x);
    cur.share = 0;
    if (SPLIT) {
      // The first SHARED items have a cluster each, the others a CTA: so many that all clusters run at once
      index /= parts;
      int shared = nslots * p.kv_heads;
      if (sorted) {
        const int items = p.kv_heads * static_cast<int>(__reduce_add_sync(0xffffffffu, pairs));
        const int lengthy = p.kv_heads * static_cast<int>(__reduce_add_sync(0xffffffffu, mine.nk >= MIN_SHARED ? pairs : 0));
        shared = min(items <= fit ? items : max(parts * fit - items, 0) / (parts - 1), lengthy);
      }
      cur.share = index < shared;
      if (!cur.share) index = shared + (index - shared) * parts + part;
    }
    if (!find(index, cur)) next_item(cur);
    uint32_t q_count[2] = {0, 0}, loads = 0;  // so far
    for (uint32_t k = 0;; ++k) {
      const int ib = k & 1;
      if (*abort_flag) ok = false;
      if (!__shfl_sync(0xffffffffu, lane == 0 ? wait_item(&bars->item_empty[ib], ((k >> 1) & 1) ^ 1, 8) : true, 0)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) cur.kvh = -1;
      if (lane == 0) {
        bars->item[ib] = cur;
        mbar_arrive(&bars->item_full[ib]);
      }
      __syncwarp();
      if (cur.kvh < 0) break;
      // a tile of Q: the box (64 dims, g heads, tpt tokens), rows token-major; rows of the tile past g tpt stay
      // as they are and are never stored.  Only for a tile that has units here: its product's end is what the
      // softmax warps wait for before they write over Q's memory, so no copy may be left that nothing waits for.
      for (int x = 0; x < cur.tiles; ++x) {
        if (cur.nu[x] == 0) continue;
        ok = ok && mbar_wait_warp(&bars->q_empty[x], (q_count[x] & 1) ^ 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->q_full[x], 2 * g * tpt * 128);
          for (int hf = 0; hf < 2; ++hf)
            tma_load_3d(smem + (x ? OFF_QB : OFF_QA) + hf * HALF, &tmQ, &bars->q_full[x], hf * 64, cur.kvh * g,
                        cur.q_start + cur.t0 + x * tpt);
        }
        ++q_count[x];
      }
      Item next;
      for (int t = 0; t < 2 * cur.nloads; ++t) {
        if (t >= 2 * cur.nloads - 8 && !asked && !ended) ask();
        if (!ok) continue;
        const uint32_t sl = loads % SLOTS;
        ok = mbar_wait_warp(&bars->slot_empty[sl], ((loads / SLOTS) & 1) ^ 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
        if (!ok) continue;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->slot_full[sl], TILE_BYTES);
          const CUtensorMap* map = (t & 1) ? &tmV : &tmK;
          for (int hf = 0; hf < 2; ++hf)
            tma_load_2d(smem + OFF_SLOT + sl * TILE_BYTES + hf * HALF, map, &bars->slot_full[sl], cur.kvh * 128 + hf * 64,
                        cur.k_start + cur.key0 + (t >> 1) * TILE);
        }
        ++loads;
      }
      next_item(next);
      cur = next;
    }
    if (!ok && lane == 0) {  // the copies in flight, and an answer, land before the CTA leaves
      for (int x = 0; x < 2; ++x)
        if (q_count[x]) mbar_wait(&bars->q_full[x], (q_count[x] - 1) & 1, &no_abort, nullptr, 0);
      for (uint32_t t = loads < SLOTS ? 0 : loads - SLOTS; t < loads; ++t)
        mbar_wait(&bars->slot_full[t % SLOTS], (t / SLOTS) & 1, &no_abort, nullptr, 0);
      if (asked) mbar_wait(&bars->claim_full, claims & 1, &no_abort, nullptr, 0);
    }
  } else if (warp <= 2) {
    if (lane == 0) {
      // ---- the MMAs of tile x (descriptors as 32-bit low words over a common high word)
      const int x = warp - 1;
      const uint32_t dhi = static_cast<uint32_t>(sdesc_sw128(0, 16, 1024) >> 32);
      const uint32_t qlo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + (x ? OFF_QB : OFF_QA)), 16, 1024));
      const uint32_t klo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + OFF_SLOT), 16, 1024));    // K-major
      const uint32_t vlo = static_cast<uint32_t>(sdesc_sw128(smem_u32(smem + OFF_SLOT), HALF, 1024));  // MN-major
      const uint32_t s_tm = tmem + x * 128, o_tm = tmem + 256 + x * 128;
      uint32_t base = 0, units = 0, q_count = 0;  // loads and this tile's units of the items before
      auto slot_of = [&](int t) { return (base + t) % SLOTS; };
      auto issue_s = [&](int u) {
        const uint32_t k = klo + (slot_of((u >> 1) * 2) * TILE_BYTES + (u & 1) * UNIT * 128) / 16;
        const uint32_t d = s_tm + ((units + u) & 1) * UNIT;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t o = ((kk >> 2) * HALF + (kk & 3) * 32) / 16;
          umma_ss_lo(d, qlo + o, k + o, dhi, IDESC_S, kk ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int u) {
        const uint32_t v = vlo + (slot_of((u >> 1) * 2 + 1) * TILE_BYTES + (u & 1) * UNIT * 128) / 16;
        const uint32_t a = s_tm + ((units + u) & 1) * UNIT;
#pragma unroll
        for (int kk = 0; kk < UNIT / 16; ++kk)
          umma_ts_lo(o_tm, a + kk * 8, v + kk * 2048 / 16, dhi, IDESC_PV, (u > 0 || kk) ? 1u : 0u);
      };
      auto wait_load = [&](int t) {
        return mbar_wait(&bars->slot_full[slot_of(t)], ((base + t) / SLOTS) & 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
      };
      bool ok = true;
      for (uint32_t k = 0;; ++k) {
        const int ib = k & 1;
        if (!wait_item(&bars->item_full[ib], (k >> 1) & 1)) break;
        const int n = bars->item[ib].nu[x], nloads = bars->item[ib].nloads;
        const bool last = bars->item[ib].kvh < 0;
        mbar_arrive(&bars->item_empty[ib]);
        if (last) break;
        if (n > 0) {
          ok = ok && mbar_wait(&bars->q_full[x], q_count & 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
          ++q_count;
        }
        if (ok && n > 0 && (ok = wait_load(0))) {
          tc_fence_after();
          for (int u = 0; u < 2 && u < n; ++u) {
            issue_s(u);
            umma_commit(&bars->s_full[x][(units + u) & 1]);
          }
          umma_commit(&bars->slot_empty[slot_of(0)]);  // K_0: both its units issued
          if (n <= 2) umma_commit(&bars->q_empty[x]);
        }
        for (int u = 0; u < n && ok; ++u) {
          const int b = (units + u) & 1;
          const bool more = u + 2 < n;
          if ((u & 1) == 0 && !(ok = wait_load(2 * (u >> 1) + 1))) break;  // V(u)
          if (!(ok = mbar_wait(&bars->p_full[x][b], ((units + u) >> 1) & 1, abort_flag, status, STATUS_TIMEOUT_ATTN))) break;
          tc_fence_after();
          issue_pv(u);
          umma_commit(&bars->pv_done[x]);
          if (u + 1 == n) umma_commit(&bars->o_full[x]);
          if (more) {
            if ((u & 1) == 0 && !(ok = wait_load(2 * ((u + 2) >> 1)))) break;  // K(u + 2)
            issue_s(u + 2);
            umma_commit(&bars->s_full[x][b]);
            if (u + 3 == n) umma_commit(&bars->q_empty[x]);
          }
          // this tile's share of freeing the slots whose last reader was just issued
          if ((u & 1) == 1 || u + 1 == n) umma_commit(&bars->slot_empty[slot_of(2 * (u >> 1) + 1)]);   // V(u)
          if (more && ((u & 1) == 1 || u + 3 == n)) umma_commit(&bars->slot_empty[slot_of(2 * ((u + 2) >> 1))]);
        }
        // the loads only the other tile reads: this tile's share once each has landed
        for (int t = 2 * ((n + 1) / 2); t < 2 * nloads && ok; ++t) {
          if (!(ok = wait_load(t))) break;
          umma_commit(&bars->slot_empty[slot_of(t)]);
        }
        base += 2 * nloads;
        units += n;
      }
      umma_commit(&bars->done[x]);  // every MMA queued above has finished before TMEM is released
      mbar_wait(&bars->done[x], 0, &no_abort, nullptr, 0);
    }
  } else {
    // ---- softmax: tile x, TMEM lane quarter wq, row r of the tile
    const int x = (warp - 3) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const int tok = r / g;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + x * 128;
    const uint32_t o_addr = tmem + lane_off + 256 + x * 128;
    const uint64_t sc2 = f2(p.scale_log2, p.scale_log2);
    // the two tiles' exponentials take turns on each scheduler (attention.cu); tile a's turns end with its
    // last unit, which is never after tile b's
    const uint32_t my_turn = (x ? 5u : 1u) + static_cast<uint32_t>(wq);
    const uint32_t other_turn = (x ? 1u : 5u) + static_cast<uint32_t>(wq);
    uint32_t units = 0, o_count = 0;  // of the items before
    bool ok = true;
    const bool wide = ((reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(2 * p.ld_out)) & 31) == 0;
    for (uint32_t k = 0;; ++k) {
      const int ib = k & 1;
      if (!__shfl_sync(0xffffffffu, lane == 0 ? wait_item(&bars->item_full[ib], (k >> 1) & 1) : true, 0)) break;
      const Item& it = bars->item[ib];
      const int kvh = it.kvh, n = it.nu[x], n_a = it.nu[0], tiles = it.tiles, delta = it.delta, nq = it.nq, it_key0 = it.key0;
      const int t = it.t0 + x * tpt + tok, q_start = it.q_start, k_start = it.k_start;  // t: token within the sequence
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->item_empty[ib]);
      if (kvh < 0) break;
      const bool live = tok < tpt && t < nq && x < tiles;
      const int lim = live ? t + delta - it_key0 : n * UNIT;  // last visible key from KEY0 on (< 0: none)
      float m = -INFINITY, lsum = 0.f;
      const int turns = tiles == 2 ? n_a : 0;
      if (turns > 0 && x == 1) asm volatile("bar.arrive %0, 64;" ::"r"(other_turn) : "memory");  // tile a goes first
      for (int u = 0; u < n; ++u) {
        const int b = (units + u) & 1;
        ok = ok && mbar_wait_uniform(&bars->s_full[x][b], ((units + u) >> 1) & 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
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
            ok = mbar_wait_uniform(&bars->pv_done[x], (units + u - 1) & 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
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
        {  // log2 of P, before the turn: what is left for it is the exponentials
          const uint64_t nm2 = f2(nm, nm);
#pragma unroll
          for (int i = 0; i < UNIT; i += 2) f2_split(ffma2(f2(s[i], s[i + 1]), sc2, nm2), s[i], s[i + 1]);
        }
        if (u < turns) asm volatile("bar.sync %0, 64;" ::"r"(my_turn) : "memory");
        uint32_t pk[UNIT / 2];  // P as 16-bit pairs: key 2c and 2c+1 in column c
        if (ok) {
          uint64_t ps2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
          for (int c8 = 0; c8 < UNIT / 8; ++c8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e0 = fast_exp2(s[c8 * 8 + 2 * i]), e1 = fast_exp2(s[c8 * 8 + 2 * i + 1]);
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
      units += n;
      if (SPLIT && it.share) {
        // ---- the join of a cluster's parts.  Every CTA leaves its O (fp32) and (m, l) over Q's and the ring's memory
        // (16 bytes i of row j at i ^ (j % 32)); then each takes a share of the rows, a warp 32 / parts of them.
        if (n > 0) ok = ok && mbar_wait_uniform(&bars->o_full[x], 0, abort_flag, status, STATUS_TIMEOUT_ATTN);
        tc_fence_after();
        asm volatile("bar.sync 9, 256;" ::: "memory");  // the softmax warps': both tiles' MMAs are done
        float2* const ml = reinterpret_cast<float2*>(smem + OFF_SLOT + 2 * TILE_BYTES);
        {
          float4* const mine = reinterpret_cast<float4*>(smem + (x * TILE + r) * 512);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t rr[32];
            if (n > 0 && ok) {
              tmem_ld32(o_addr + c * 32, rr);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) rr[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              mine[(c * 8 + i) ^ lane] = make_float4(__uint_as_float(rr[4 * i]), __uint_as_float(rr[4 * i + 1]),
                                                     __uint_as_float(rr[4 * i + 2]), __uint_as_float(rr[4 * i + 3]));
          }
          ml[x * TILE + r] = make_float2(m, lsum);
        }
        cluster_sync();
        const int shift = 31 - __clz(parts), row0 = (part * 8 + warp - 3) * (32 >> shift);  // the warp's first row
        // a lane a (row, part): its weight 2^(m_c - M) / l, and of the first lanes each a row: where it goes
        float weight;
        {
          const float2 y = ld_cluster_f2(mapa_shared(ml + row0 + (lane >> shift), lane & (parts - 1)));
          float mx = y.x;
          for (int o = 1; o < parts; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          weight = fast_exp2(y.x - (mx == -INFINITY ? 0.f : mx));
          float l = weight * y.y;
          for (int o = 1; o < parts; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          weight = l == 0.f ? 0.f : weight / l;
        }
        const int row = row0 + lane, y = row / TILE, rj = row - y * TILE, tj = rj / g, token = it.t0 + y * tpt + tj;
        const bool valid = lane < (32 >> shift) && y < tiles && tj < tpt && token < nq;
        const int head = kvh * g + rj - tj * g;
        const unsigned rows_mask = __ballot_sync(0xffffffffu, valid);
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {  // 16 of the warp's 32 pieces at a time
          float4 z[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = row0 + ((b * 16 + i) >> shift);
            z[i] = ld_cluster_f4(mapa_shared(smem + j * 512 + ((lane ^ (j & 31)) << 4), i & (parts - 1)));
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float w = __shfl_sync(0xffffffffu, weight, b * 16 + i);
            z[i] = make_float4(w * z[i].x, w * z[i].y, w * z[i].z, w * z[i].w);
          }
          // the sums over 2, 4 or 8 parts move to the front
#pragma unroll
          for (int s2 = 1; s2 < 8; s2 *= 2)
            if (s2 < parts)
#pragma unroll
              for (int i = 0; i < 8 / s2; ++i)
                z[i] = make_float4(z[2 * i].x + z[2 * i + 1].x, z[2 * i].y + z[2 * i + 1].y, z[2 * i].z + z[2 * i + 1].z,
                                   z[2 * i].w + z[2 * i + 1].w);
          const int k0 = (b * 16) >> shift;
          unsigned bad = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = k0 + i, to = __shfl_sync(0xffffffffu, token, k), h = __shfl_sync(0xffffffffu, head, k);
            if (i < (16 >> shift) && ((rows_mask >> k) & 1)) {
              const float4 o = z[i];
              reinterpret_cast<uint2*>(out + static_cast<long long>(q_start + to) * p.ld_out + h * 128)[lane] =
                  make_uint2(pack16<F16>(o.x, o.y), pack16<F16>(o.z, o.w));
              if (!(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w))) bad |= 1u << k;
            }
          }
          bad = __reduce_or_sync(0xffffffffu, bad);
          while (bad) {
            const int k = __ffs(bad) - 1, to = __shfl_sync(0xffffffffu, token, k), h = __shfl_sync(0xffffffffu, head, k);
            bad &= bad - 1;
            const long long seen = min(nq, it.t0 + ((row0 + k) / TILE + 1) * tpt) + delta;  // by the tile's last row
            const long long end = min((seen + UNIT - 1) / UNIT * UNIT, p.kv_rows - k_start), kr = k_start;
            mend_row<F16>(static_cast<const uint16_t*>(p.q) + static_cast<long long>(q_start + to) * p.ld_q + h * 128,
                          static_cast<const uint16_t*>(p.k) + kr * p.ld_k + kvh * 128, p.ld_k,
                          static_cast<const uint16_t*>(p.v) + kr * p.ld_v + kvh * 128, p.ld_v, to + delta,
                          static_cast<int>(end) - 1, p.scale_log2,
                          out + static_cast<long long>(q_start + to) * p.ld_out + h * 128);
            __syncwarp();
          }
        }
        cluster_sync();  // no CTA leaves while another reads its parts
        joined = true;
        break;  // a cluster has one item
      }
      const int head = kvh * g + r - tok * g;
      uint16_t* dst = out + static_cast<long long>(q_start + t) * p.ld_out + head * 128;
      if (n > 0) {
        ok = ok && mbar_wait_uniform(&bars->o_full[x], o_count & 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
        ++o_count;
        if (ok) {
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
              uint32_t w[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = pack16<F16>(o[2 * i], o[2 * i + 1]);
              // a row a lane: half the lines of 16-byte stores (30 sequences of 300: 58.3 us, 62.1)
              if (wide) {
                st_global_32(dst + c * 32, w);
                st_global_32(dst + c * 32 + 16, w + 8);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  reinterpret_cast<uint4*>(dst + c * 32)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
              }
            }
          }
          tc_fence_before();  // O is read before the next item's first P lets an MMA write it
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
  }
  if (SPLIT && !joined) {  // the join's barriers are all threads', whatever ended their work
    __syncwarp();
    cluster_sync();
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// a launch of ITEMS clusters of PARTS CTAs that may start while the kernel before it ends
struct PackedLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  PackedLaunch(unsigned items, int parts, cudaStream_t st) {
    cfg.gridDim = dim3(items * parts);
    cfg.blockDim = dim3(PK_THREADS);
    cfg.dynamicSmemBytes = PK_SMEM;
    cfg.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = parts;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = parts > 1 ? 2 : 1;
  }
  PackedLaunch(const PackedLaunch&) = delete;
};

int packed_prepare(int (&fit)[3]) {
  for (auto* kernel : {k_packed<false, false>, k_packed<true, false>, k_packed<false, true>, k_packed<true, true>}) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PK_SMEM);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  for (int i = 0; i < 3; ++i) {
    PackedLaunch l(1, 2 << i, nullptr);
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&fit[i], k_packed<false, true>, &l.cfg);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
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
  const long long nslots = (a.rows - 1) / (2 * tpt) + a.nseq, items = nslots * a.kv_heads;  // at most
  if (items > 0x7fffffffll) return -1;
  // CTAs a cluster.  Its launch and join cost about 5 us, so it has to have keys enough to share, and all clusters
  // run at once (74 of 2, 33 of 4, 15 of 8).  us at 1, 2, 4 and 8 CTAs an item (32 heads over 8, bf16):
  //   64 rows (8 items)    over 512 keys:  15 15 14 16    over  768: 18 17 16 16    over 16384: 247 134  73  46
  //   192 rows (24 items)  over 512 keys:  15 15 15       over  768: 19 18 17       over  8192: 128  73  45
  //   512 rows (64 items)  over 512 keys:  15 16          over 1024: 23 20          over  8192: 128  75
  // Up to twice the clusters of 2, some items are shared; with one sequence, whose items are alike, that gains
  // nothing (1024 rows over 1100 keys: 24 us either way), with several it does when their keys differ (300, 77,
  // 512 and 9 rows over 4100, 900, 513 and 5 keys, 28 heads over 4: 68 us alone, 44 so).
  const long long keys = a.kv_rows / a.nseq;
  const int parts = keys < MIN_SHARED ? 1 : items <= a.fit[2] ? 8 : items <= a.fit[1] ? 4
                    : items <= (a.nseq > 1 && a.nseq <= 32 ? 2 : 1) * a.fit[0] ? 2 : 1;
  const int fit = parts > 1 ? a.fit[parts == 8 ? 2 : parts == 4 ? 1 : 0] : 0;
  const PackedLaunch l(static_cast<unsigned>(parts > 1 && items > fit ? fit : items), parts, st);
  auto* const kernel = parts > 1 ? (a.f16 ? k_packed<true, true> : k_packed<false, true>)
                                 : (a.f16 ? k_packed<true, false> : k_packed<false, false>);
  return static_cast<int>(cudaLaunchKernelEx(&l.cfg, kernel, tq, tk, tv, a, tpt, static_cast<int>(nslots), fit, d_status));
}

}  // namespace exn
