// attn_cache.cu -- keys and values held in 8 bits, and attention over them,
// head dim 128 (no counterpart in the reference: illatio keeps its keys and
// values in fp32 for the one call, src/encoder.lisp:143-183).
//
// A page holds 64 positions of one sequence; for each key/value head it has
// codes int8 [64][128] and one scale.  The scale is a power of two, 2^e with
// the smallest e >= -126 such that max |x| <= 127 2^e over what the page has
// held so far.  A code is x / 2^e rounded to the nearest integer (half to
// even), so a value is off by at most 2^e / 2; when a later token makes e grow
// by d, the page's codes become code / 2^d rounded the same way, and the sum of
// all such errors stays below 2^e.  Powers of two make every step but those
// roundings exact, and code * 2^e is exactly a bf16 number (8 significant
// bits): what the cache stands for does not depend on who reads it.  A page
// that is given an infinity or a NaN gets the scale NaN and makes NaN of what
// is read from it until it starts anew at its first position.
#include <atomic>
#include <chrono>

#include "exn_device.cuh"
#include "exn_internal.h"

namespace exn {

int make_tmap(CUtensorMap* m, CUtensorMapDataType type, const void* base, int rank, const uint64_t* dims,
              const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle);

namespace {

constexpr int PAGE_BYTES = kPage * 128;  // one head's codes of a page

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

// the smallest e >= -126 with amax <= 127 2^e, amax finite and >= 0
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 127;     // floor(log2 amax) of a normal number
  const uint32_t mant = bits & 0x7fffffu;               // 127 = 2^6 * 1.984375, mantissa 0x7e0000
  const int r = e - 6 + (mant > 0x7e0000u ? 1 : 0);
  return r < -126 ? -126 : r;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// 2^e of a whole number -127 (0 then) .. 127: its exponent is in the low bits of a float whose unit is 1
__device__ __forceinline__ float pow2_of(float e) { return __uint_as_float(__float_as_uint(e + 0x1.8000fep23f) << 23); }

__device__ __forceinline__ int to_code(float x, float top) { return __float2int_rn(fminf(fmaxf(x, -top), top)); }

// The rows of a call that fall into one page, by the page's slot: sequence s owns the slots from
// floor(start_s / 64) + 2 s on, of which its rows, consecutive positions, touch at most ceil(count / 64) + 1.
struct PageRows {
  int s, page_i;    // the sequence (-1: none) and its page
  int lo, hi;       // the page's rows of this call: lo .. hi - 1
  long long row0;   // the row of the page's position 0 (below 0 where the call starts inside the page)
};
// All threads; FOUND is shared by the block.  From the first sequence whose offsets decrease on there are none: a
// later one could own rows and slots of an earlier one, so that two threads would fill FOUND.  Before it the
// sequences' slots are disjoint.
__device__ __forceinline__ void find_page(const int* offsets, const int* lens, int nseq, long long rows, int slot,
                                          PageRows* found, int* status) {
  __shared__ int decrease;
  if (threadIdx.x == 0) {
    found->s = -1;
    decrease = nseq;
  }
  __syncthreads();
  PageRows mine = {-1, 0, 0, 0, 0};
  for (int s = threadIdx.x; s < nseq; s += blockDim.x) {
    const int a = offsets[s], b = offsets[s + 1], len = lens[s];
    if (b < a) atomicMin(&decrease, s);
    if (a < 0 || b < a || b > rows || len < b - a) {
      if (blockIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      continue;
    }
    if (b == a || mine.s >= 0) continue;
    const int pos0 = len - (b - a), p0 = pos0 / kPage, p1 = (len - 1) / kPage;
    const long long i = slot - (a / kPage + 2ll * s);
    if (i < 0 || i > p1 - p0) continue;
    mine.s = s;
    mine.page_i = p0 + static_cast<int>(i);
    const long long base = static_cast<long long>(mine.page_i) * kPage;
    mine.lo = static_cast<int>(max(pos0 - base, 0ll));
    mine.hi = static_cast<int>(min(len - base, static_cast<long long>(kPage)));
    mine.row0 = a + base - pos0;
  }
  __syncthreads();
  if (mine.s >= 0 && mine.s < decrease) *found = mine;
  __syncthreads();
}

// ---- write: one block = one page touched by the call's rows, one key/value head, K or V; 16 threads a row of
// 128 values.  Long prompts are bound by the bytes, 2 in and 1 out a value (6360 rows of 8 heads: 7.6 us, 5.1
// TB/s); single tokens (64: 4.6 us) by the chain of dependent loads (offsets and lengths; the rows and the
// table's entry; the page's scale; its codes, when the scale grows).
template <bool F16>
__global__ void __launch_bounds__(128) k_cache_write(const CacheArgs c, const int* __restrict__ offsets,
                                                     long long rows, const uint16_t* __restrict__ k, long long ld_k,
                                                     const uint16_t* __restrict__ v, long long ld_v, int* status) {
  __shared__ PageRows at;
  __shared__ uint32_t red[4];
  const int slot = blockIdx.x / (2 * c.kv_heads), h = blockIdx.x % (2 * c.kv_heads) >> 1;
  griddep_wait();
  griddep_launch();
  find_page(offsets, c.lens, c.nseq, rows, slot, &at, status);
  if (at.s < 0) return;
  const int page = at.page_i < c.table_ld ? c.table[static_cast<long long>(at.s) * c.table_ld + at.page_i] : -1;
  const int lo = at.lo, hi = at.hi;
  const bool is_v = blockIdx.x & 1;
  const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4;  // 8 values at 8 sub of rows r0, r0 + 8, ..
  const long long ld = is_v ? ld_v : ld_k;
  const uint16_t* src = (is_v ? v : k) + at.row0 * ld + h * 128 + sub * 8;

  uint4 x[8];
  uint32_t mag = 0;  // the largest magnitudes of the even and odd values, as bits: their order is that of the values
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 8 * i;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (r >= lo && r < hi) x[i] = __ldg(reinterpret_cast<const uint4*>(src + r * ld));
  }
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    return;
  }
  const long long head = static_cast<long long>(page) * c.kv_heads + h;
  int8_t* dst = (is_v ? c.v : c.k) + head * PAGE_BYTES + sub * 8;
  float* scale = (is_v ? c.v_scale : c.k_scale) + head;
  const float before = lo > 0 ? *scale : 0.f;  // what the page holds already (none when it starts anew)
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) mag = __vmaxu2(mag, reinterpret_cast<const uint32_t*>(&x[i])[j] & 0x7fff7fffu);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mag = __vmaxu2(mag, __shfl_xor_sync(0xffffffffu, mag, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mag;
  __syncthreads();
  mag = __vmaxu2(__vmaxu2(red[0], red[1]), __vmaxu2(red[2], red[3]));
  const float amax = unpack16<F16>(max(mag & 0xffffu, mag >> 16)).x;
  const bool poisoned = !(amax < INFINITY) || before != before;  // infinite or NaN
  const float mine = pow2(scale_exponent(poisoned ? 0.f : amax));
  const float now = fmaxf(mine, before);
  const float inv = 1.f / now;  // exact: a power of two between 2^-122 and 2^126
  const float top = now == (F16 ? 0x1p10f : 0x1p122f) ? 63.f : 127.f;  // 64 of the type's largest scale are infinite
  if (lo > 0 && !poisoned && now > before) {  // the codes that are there, in the larger unit
    const float f = before * inv;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + 8 * i;
      if (r < lo) {
        uint2* p = reinterpret_cast<uint2*>(dst + r * 128);
        uint2 w = *p;
        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t n = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int q = to_code(static_cast<float>(static_cast<int8_t>(u[j] >> (8 * b))) * f, top);
            n |= (static_cast<uint32_t>(q) & 0xffu) << (8 * b);
          }
          u[j] = n;
        }
        *p = w;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 8 * i;
    if (r >= lo && r < hi) {
      uint32_t u[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 a = unpack16<F16>(reinterpret_cast<const uint32_t*>(&x[i])[2 * j]);
        const float2 b = unpack16<F16>(reinterpret_cast<const uint32_t*>(&x[i])[2 * j + 1]);
        float f[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = fmaf(f[e], inv, 0x1.8p23f);  // rounded to an integer, which is then the low bits
          if (top != 127.f) f[e] = fminf(fmaxf(f[e], 0x1.8p23f - top), 0x1.8p23f + top);
        }
        const uint32_t n = poisoned ? 0u : __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040),
                                                       __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040), 0x5410);
        u[j] = n;
      }
      *reinterpret_cast<uint2*>(dst + r * 128) = make_uint2(u[0], u[1]);
    }
  }
  if (threadIdx.x == 0) *scale = poisoned ? __uint_as_float(0x7fffffffu) : now;
}

// ---- read: the same blocks; code * scale in 16 bits (exact in bf16; rounded once where fp16's range
// ends).  DENSE: every position, to row s * table_ld * 64 + position.  Bound by the bytes, 1 in, 2 out
// (7157 rows of 8 heads: 7.0 us, 6.3 TB/s).
template <bool F16, bool DENSE>
__global__ void __launch_bounds__(128) k_cache_read(const CacheArgs c, const int* __restrict__ offsets,
                                                    long long rows, uint16_t* __restrict__ k, long long ld_k,
                                                    uint16_t* __restrict__ v, long long ld_v, int* status) {
  __shared__ PageRows found;
  const int slot = blockIdx.x / (2 * c.kv_heads), h = blockIdx.x % (2 * c.kv_heads) >> 1;
  griddep_wait();
  griddep_launch();
  PageRows at;
  if (DENSE) {
    at.s = slot / c.table_ld;
    at.page_i = slot - at.s * c.table_ld;
    const int len = c.lens[at.s];
    if (len < 0 || len > static_cast<long long>(c.table_ld) * kPage) {
      if (at.page_i == 0 && threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      return;
    }
    if (len <= at.page_i * kPage) return;
    at.lo = 0;  // the last page whole: the rows behind the sequence's last are then finite, as its codes are
    at.hi = kPage;
    at.row0 = static_cast<long long>(slot) * kPage;
  } else {
    find_page(offsets, c.lens, c.nseq, rows, slot, &found, status);
    at = found;
    if (at.s < 0) return;
  }
  const int page = at.page_i < c.table_ld ? c.table[static_cast<long long>(at.s) * c.table_ld + at.page_i] : -1;
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    return;
  }
  const bool is_v = blockIdx.x & 1;
  const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const long long head = static_cast<long long>(page) * c.kv_heads + h;
  const int8_t* src = (is_v ? c.v : c.k) + head * PAGE_BYTES + sub * 8;
  const float scale = (is_v ? c.v_scale : c.k_scale)[head];
  const long long ld = is_v ? ld_v : ld_k;
  uint16_t* dst = (is_v ? v : k) + at.row0 * ld + h * 128 + sub * 8;
  uint2 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 8 * i;
    if (r >= at.lo && r < at.hi) w[i] = *reinterpret_cast<const uint2*>(src + r * 128);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 8 * i;
    if (r < at.lo || r >= at.hi) continue;
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[i]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = u[j >> 1] >> (16 * (j & 1));
      o[j] = pack16<F16>(static_cast<float>(static_cast<int8_t>(pair)) * scale,
                         static_cast<float>(static_cast<int8_t>(pair >> 8)) * scale);
    }
    *reinterpret_cast<uint4*>(dst + r * ld) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---- attention of a few rows over the codes
//
// An item is a tile of up to 8 NT query rows (tokens times the query heads that read one key/value head)
// of one sequence; its work is the sequence's half pages ("spans", 32 positions) and SETUP more for what an
// item costs by itself.  The work of all items, laid end to end, is cut into equal parts, one a CTA, so a
// launch is one wave whatever the lengths: a long sequence is shared by many CTAs, short ones share a CTA.
// In a CTA one warp brings the data and the others compute: the producer finds the CTA's part of the work,
// turns each item's rows of q into the MMA's operand (but the first's, whose readers wait) and streams the spans with TMA, dealt out to the
// other warps in turn, through a ring of 4 KB tiles each (K_0 V_0 K_1 ..; 128-byte swizzle, so that the
// reads below touch every bank once); it runs ahead from one item into the next.  Each computing warp has
// its own running maximum, sum and output, joined through shared memory at the item's end.  An item that is
// cut leaves each CTA's joined part in the workspace and counts it; the CTA whose part is the last (nobody
// waits) adds the parts in their order, so the bits do not depend on who it was.  The count is kept under
// the launch's tag, a number that no other launch of the process has, so whatever the workspace held before
// is not taken for one.
//
// Bound by the codes' bytes (a code takes part in 4 g c operations) as long as the instructions keep up: 64
// tokens over 500 to 8192 positions each, 334 MB, take 66.5 us (5.0 TB/s; 6.2 from the first copy to the last), one
// over 130001, 266 MB, 56 us.  One over 1001 takes 9.1 us, all latency: launch 1.4, lengths and cut 1.8, the
// first span 2.7, the join over memory 3.
// A byte permute, a logical operation and a paired fp16 one each take a scheduler two clocks a warp, an
// MMA eight, so what turns codes into operands is what counts:
//   * codes are the 16-row operand and the queries the 8 columns: S^T = K Q^T, O^T = V^T P^T, so 8
//     rows of queries waste nothing;
//   * K's codes are multiplied as they are (m16n8k32, s8): a row of q is two int8 numbers, q = 2^a (hi +
//     lo / 256) with 2^a the smallest power of two that |q| <= 127 2^a allows.  The sums are exact; q
//     itself is, for elements of 1/128 (bf16) or 1/16 (fp16) of the row's largest M and more, and off by
//     at most 2^a / 512 <= M / 32512 below.  Over 128 codes of up to 127 that moves a score by no more than M / 2
//     of K's scale, which is what K's own rounding may do in one element;
//   * V's codes become fp16 (m16n8k16), exactly: ldmatrix.trans brings a position pair's codes of two
//     dims into one register, from which 1024 + (code + 128) is 0x6400 | byte, less 1152;
//   * what multiplies them is P' = P 2^(ev - u) in fp16, P the fp32 softmax weight, 2^ev the page's scale and
//     2^u the unit of the row's sums, a power of two that follows the row's largest P 2^ev: P' stays
//     between 1 and 2^14 for it, so what fp16 drops (P' < 2^-25) is 2^-25 of the row's largest product of a
//     weight and a scale, whatever the scales of the pages are.  The sums are rescaled only when the row
//     maximum grows by more than 2^8 or P' would leave that range;
//     The tensor core cuts its sums where other units round, so a warp's over n half pages come out low by
//     about n 2^-24 of themselves (2^20 half pages over five warps: 1.1 %): 2^-11 and more only from 2^13 a warp on,
//     which is a call over 100 GB of codes;
//   * P^T turns from the first product's layout to the second's with movmatrix.
constexpr int SPAN = 32;                  // positions a warp takes at a time
constexpr int SPAN_BYTES = SPAN * 128;
constexpr int SETUP = 12;                 // what an item costs besides its spans, in spans
constexpr int MIN_PART = 16 + SETUP;      // the least work worth a CTA that may take several items

// Tiles of 8 rows (NT 1): two CTAs of 5 + 1 warps an SM, 168 registers a thread (20 bytes spilled); of 16 rows,
// whose sums take twice the registers, one of 7 + 1, 255 (32 bytes)
template <int NT>
struct AttendCfg {
  static constexpr int WARPS = NT == 1 ? 5 : 7, CTAS = NT == 1 ? 2 : 1, ROWS = 8 * NT, THREADS = (WARPS + 1) * 32;
  static constexpr int SLOTS = 4;
  static constexpr int RING = WARPS * SLOTS * SPAN_BYTES, JOIN = WARPS * ROWS * 512;
  static constexpr int SMEM = RING + JOIN + 1024;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// d = a b + the integer whose bits are the float 1.5 * 2^23: the float of d's bits less that is the product
__device__ __forceinline__ void mma16832_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0x4b400000));
}
__device__ __forceinline__ void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two of four biased codes (code + 128), bytes 0 and 2 or 1 and 3, as fp16: 1024 + byte - 1152, exact
__device__ __forceinline__ uint32_t v_pair(uint32_t u, uint32_t sel) {
  const uint32_t h = __byte_perm(u, 0x64646464u, sel);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&x);
}
constexpr uint32_t EVEN = 0x4240, ODD = 0x4341;
// four 8 x 8 matrices of 16-bit elements, transposed; a lane's address is a row of one of them
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void fence_acq_rel() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

// The counts of an item's parts, tag + parts so far.  Before a launch there is 0, what the last part leaves, or
// anything that is not the launch's tag.  The CTA that the item begins in raises it to the tag when it
// starts; a part that finds no tag all the same (it came earlier, or there was something larger) puts it
// there.
__device__ __forceinline__ bool tagged(unsigned long long v, unsigned long long tag) { return (v & ~0xffffull) == tag; }
__device__ __forceinline__ void start_count(unsigned long long* at, unsigned long long tag) {
  asm volatile("red.relaxed.gpu.global.max.u64 [%0], %1;" ::"l"(at), "l"(tag) : "memory");
}
// one more part: how many there were before
__device__ __forceinline__ int count_part(unsigned long long* at, unsigned long long tag) {
  unsigned long long v = atomicAdd(at, 1ull);
  while (!tagged(v, tag)) {  // a few times at most: only the item's parts change it
    const unsigned long long got = atomicCAS(at, v + 1, tag + 1);
    if (got == v + 1) return 0;
    v = tagged(got, tag) ? atomicAdd(at, 1ull) : got - 1;
  }
  return static_cast<int>(v & 0xffffull);
}

// TX more bytes expected in the phase at hand; no arrival
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t tx) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(tx) : "memory");
}

// whether the phase of parity PARITY is complete; never waits
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// How a launch's work is cut, and its workspace
struct AttendPlan {
  int nt;                     // tiles of 8 nt rows
  int hpt, head_tiles, tpt;   // heads and tokens a tile, tiles of a key/value head's query heads
  int ctas;
  unsigned long long tag;     // its low 16 bits are 0
  // [ctas]: the parts of the item that begins in the CTA's work and goes on behind it, counted
  unsigned long long* count;
  // part 2 c: of the item that began before CTA c's work, 2 c + 1: of the one that goes on behind it
  float* part;                // [2 ctas][ROWS][132]: o unnormalised, m, l
};

// A CTA's part of an item
struct Seg {
  int row0, tok, head0, nh;   // first row, tokens, first head, heads
  int kvh, pos0;              // key/value head, position of the first row
  int sp0, n, spans, item;    // spans sp0 .. sp0 + n - 1 of the item's; where it begins in the work
};

template <int NT>
struct AttendShared {
  using C = AttendCfg<NT>;
  uint64_t full[C::WARPS][C::SLOTS], empty[C::WARPS][C::SLOTS];  // the rings
  uint64_t seg_full[2], seg_empty[2];
  Seg seg[2];                                    // n 0: no more
  uint32_t q[2][2][C::ROWS][32];                 // [segment][hi, lo][row]: 128 codes
  float q_scale[2][C::ROWS];                     // 2^a scale log2(e)
  float4 meta[C::WARPS][2];                      // of a warp's span: K's and V's scale, first position (bits)
  float m[C::WARPS][C::ROWS], l[C::WARPS][C::ROWS];
  int part_len, lead, taken, abort_word;
};

// A row of q, four dims a lane, as 2^a (hi + lo / 256) into row R of segment buffer B.  By a whole warp.
template <bool F16, int NT>
__device__ __forceinline__ void put_query(AttendShared<NT>& sh, int b, int r, uint2 w, float scale_log2) {
  const int lane = threadIdx.x & 31;
  const uint32_t mag = __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);  // magnitudes order as their bits do
  const float mx = unpack16<F16>(__reduce_max_sync(0xffffffffu, max(mag & 0xffffu, mag >> 16))).x;
  const bool bad = !(mx < INFINITY);
  const int e = scale_exponent(bad ? 0.f : mx);
  const float inv = pow2(-e);
  const float2 v01 = unpack16<F16>(w.x), v23 = unpack16<F16>(w.y);
  const float v[4] = {v01.x, v01.y, v23.x, v23.y};
  uint32_t hi[4], lo[4];  // in the low bits of floats near 1.5 * 2^23, whose unit is 1
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = v[i] * inv, h = __fadd_rd(x + 0x1.01p-1f, 0x1.8p23f);  // hi: lo is then -128 .. 127 without a clamp
    hi[i] = __float_as_uint(h);
    lo[i] = __float_as_uint(fmaf(x - (h - 0x1.8p23f), 256.f, 0x1.8p23f));
  }
  sh.q[b][0][r][lane] = __byte_perm(__byte_perm(hi[0], hi[1], 0x0040), __byte_perm(hi[2], hi[3], 0x0040), 0x5410);
  sh.q[b][1][r][lane] = __byte_perm(__byte_perm(lo[0], lo[1], 0x0040), __byte_perm(lo[2], lo[3], 0x0040), 0x5410);
  if (lane == 0) sh.q_scale[b][r] = bad ? __uint_as_float(0x7fffffffu) : scale_log2 * pow2(e);  // not finite: NaN
}

// ---- the producer warp
template <bool F16, int NT>
__device__ __forceinline__ void attend_produce(const CUtensorMap* tmK, const CUtensorMap* tmV, const CacheAttnArgs& p,
                                               const AttendPlan& plan, AttendShared<NT>& sh, uint8_t* ring, int* status) {
  using C = AttendCfg<NT>;
  constexpr int ROWS = C::ROWS, WARPS = C::WARPS, SLOTS = C::SLOTS;
  const int lane = threadIdx.x & 31;
  const int kv = p.c.kv_heads, g = p.heads / kv, per = plan.head_tiles * kv;
  volatile int* abort_flag = &sh.abort_word;

  // ---- this CTA's part of the work, [f, fend)
  auto spans_of = [](int len) { return max(1, (len + SPAN - 1) / SPAN); };
  // the items of a sequence of rows a .. b - 1; 0 for one whose numbers are out of range
  auto items_of = [&](int a, int b, int len) -> int {
    if (a < 0 || b < a || b > p.rows || len < 0 || len > static_cast<long long>(p.c.table_ld) * kPage) {
      if (blockIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      return 0;
    }
    return (plan.tpt == 1 ? b - a : (b - a + plan.tpt - 1) / plan.tpt) * per;
  };
  const int chunk = (p.c.nseq + 31) / 32;  // a run of sequences a lane
  const int s_lo = min(p.c.nseq, lane * chunk), s_hi = min(p.c.nseq, s_lo + chunk);
  long long lane_work = 0;
  int items = 0, longest = 0, start = 0, end = 0, len = 0;  // start, end, len: the lane's first sequence's
  int decrease = p.c.nseq;  // the sequences from the first whose offsets decrease on are left out
  for (bool again = true; again;) {
    const int stop = decrease;
    lane_work = 0;
    items = longest = 0;
    for (int s = s_lo; s < s_hi; ++s) {
      const int a = p.offsets[s], b = p.offsets[s + 1], l = p.c.lens[s];
      int n = items_of(a, b, l);
      if (b < a) decrease = min(decrease, s);
      if (s >= decrease) n = 0;
      items += n;
      lane_work += static_cast<long long>(n) * (spans_of(l) + SETUP);
      if (n) longest = max(longest, spans_of(l));
      if (s == s_lo) {
        start = a;
        end = b;
        len = l;
      }
    }
    decrease = __reduce_min_sync(0xffffffffu, decrease);
    again = decrease < stop;  // once more without those behind it
  }
  bool work_here = true;
  if (__any_sync(0xffffffffu, lane_work >= (1ll << 26))) {  // 2^26 spans are 512 GB of codes
    if (lane == 0) atomicOr(status, STATUS_BAD_ARG);
    work_here = false;
  }
  const int work = static_cast<int>(lane_work);
  int work_to = work, items_to = items;  // up to and with this lane's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, work_to, o), y = __shfl_up_sync(0xffffffffu, items_to, o);
    if (lane >= o) {
      work_to += x;
      items_to += y;
    }
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  const int all_work = __shfl_sync(0xffffffffu, work_to, 31), all_items = __shfl_sync(0xffffffffu, items_to, 31);
  // Equal parts of the work end to end, of at least MIN_PART; or, when the items are so few that each can have
  // CTAs of its own and the longest one's parts are no longer for it, whole CTAs an item (a span a warp at
  // least): no CTA then takes more than one item.
  int part_len = max(MIN_PART, all_work / plan.ctas + (all_work % plan.ctas ? 1 : 0));  // ALL_WORK: up to 2^31 - 1
  int stride = 0;  // an item's length when it has CTAs of its own: so many times part_len
  if (all_items > 0 && all_items <= plan.ctas) {
    const int each = min(plan.ctas / all_items, (longest + WARPS - 1) / WARPS);
    const int own = (longest + each - 1) / each;
    if (own <= part_len) {
      part_len = own;
      stride = own * each;
    }
  }
  const int lead = stride ? 0 : SETUP;
  auto item_len = [&](int spans) { return stride ? stride : spans + SETUP; };
  const long long f64 = static_cast<long long>(part_len) * blockIdx.x;
  const int total = stride ? all_items * stride : all_work;  // below 2^31: stride < longest + ctas, items <= ctas
  work_here = work_here && f64 < total;
  int f = work_here ? static_cast<int>(f64) : 0;
  const int fend = work_here ? f + min(part_len, total - f) : 0;
  int seq = s_lo, count = end - start;
  int base = stride ? (items_to - items) * stride : work_to - work;
  if (work_here) {
    const bool here = f >= base && f < base + (stride ? items * stride : work);
    if (here)
      while (true) {
        const int w = items_of(start, start + count, len) * item_len(spans_of(len));
        if (f < base + w) break;
        base += w;
        ++seq;
        start = p.offsets[seq];
        count = p.offsets[seq + 1] - start;
        len = p.c.lens[seq];
      }
    const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    seq = __shfl_sync(0xffffffffu, seq, owner);
    start = __shfl_sync(0xffffffffu, start, owner);
    count = __shfl_sync(0xffffffffu, count, owner);
    len = __shfl_sync(0xffffffffu, len, owner);
    base = __shfl_sync(0xffffffffu, base, owner);
    if (lane == 0) start_count(plan.count + blockIdx.x, plan.tag);
  }
  // the next part of an item: its description (n 0: no more), the row of the table, the positions seen
  const int* table = nullptr;
  int seen = 0;
  auto advance = [&]() -> Seg {
    Seg x = {};
    while (f < fend) {
      const int spans = spans_of(len), whole_len = item_len(spans);
      const int w = items_of(start, start + count, len) * whole_len;
      if (f >= base + w) {  // the next sequence
        base += w;
        ++seq;
        start = p.offsets[seq];
        count = p.offsets[seq + 1] - start;
        len = p.c.lens[seq];
        continue;
      }
      const unsigned idx = static_cast<unsigned>(f - base) / static_cast<unsigned>(whole_len);
      x.item = base + static_cast<int>(idx) * whole_len;  // its spans begin LEAD later
      const int f_next = min(x.item + whole_len, fend);
      x.sp0 = max(f - x.item - lead, 0);
      x.n = min(max(f_next - x.item - lead, 0), spans) - x.sp0;
      f = f_next;
      if (x.n <= 0) {  // none of its spans lie here
        x.n = 0;
        continue;
      }
      const unsigned tile = idx < static_cast<unsigned>(per) ? 0u : idx / static_cast<unsigned>(per), rest = idx - tile * per;
      const int ht = plan.head_tiles == 1 ? 0 : rest / static_cast<unsigned>(kv);
      const int t0 = static_cast<int>(tile) * plan.tpt;  // first token of the tile; token t is position t + len - count
      x.spans = spans;
      x.kvh = rest - ht * kv;
      x.row0 = start + t0;
      x.tok = min(plan.tpt, count - t0);
      x.head0 = x.kvh * g + ht * plan.hpt;
      x.nh = min(plan.hpt, g - ht * plan.hpt);
      x.pos0 = t0 + len - count;
      seen = x.pos0 + x.tok;
      table = p.c.table + static_cast<long long>(seq) * p.c.table_ld;
      break;
    }
    return x;
  };
  // page and scales of span I of a segment; a span that nothing of the tile sees or whose page is not the pool's
  // has the scale -1 and is left out
  struct Ids {
    int pid;
    float sk, sv;
  };
  auto fetch_ids = [&](const Seg& x, const int* tab, int upto, int i) -> Ids {
    Ids r = {0, -1.f, 0.f};
    if (lane < WARPS && i < x.n && (x.sp0 + i) * SPAN < upto) {
      const int id = __ldg(tab + ((x.sp0 + i) >> 1));
      if (id < 0 || id >= p.c.pages) {
        atomicOr(status, STATUS_BAD_ARG);
      } else {
        r.pid = id;
        r.sk = __ldg(p.c.k_scale + static_cast<long long>(id) * kv + x.kvh);
        r.sv = __ldg(p.c.v_scale + static_cast<long long>(id) * kv + x.kvh);
      }
    }
    return r;
  };
  // what a computing warp has to know of span SP; one that is left out lies behind every row
  auto span_meta = [](const Ids& x, int sp) {
    return make_float4(x.sk, x.sv, __int_as_float(x.sk < 0.f ? 0x7ffffff0 - SPAN : sp * SPAN), 0.f);
  };
  // a segment's rows, four dims a lane
  uint2 qw[ROWS];
  auto load_q = [&](const Seg& x) {
    int tok = 0, hd = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      qw[r] = make_uint2(0u, 0u);
      if (tok < x.tok)
        qw[r] = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + (x.row0 + tok) * p.ld_q +
                                                     (x.head0 + hd) * 128 + 4 * lane));
      if (++hd >= x.nh) {
        hd = 0;
        ++tok;
      }
    }
  };

  // lane w < WARPS serves computing warp w: spans TURN, TURN + WARPS, .. of a segment, through its ring's slot
  // SLOT next; its page numbers and scales are read a span ahead
  int turn = lane, slot = 0;
  uint32_t phase = 0, use = 0;
  Seg cur = advance();
  const int* cur_table = table;
  int cur_seen = seen;
  Ids ids = {};
  auto publish = [&](int b) {
    if (lane == 0) {
      sh.seg[b] = cur;
      sh.part_len = part_len;
      sh.lead = lead;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.seg_full[b]);
  };
  publish(0);  // the first segment's rows are turned into the operand by the computing warps, which wait anyway
  if (cur.n) {
    ids = fetch_ids(cur, cur_table, cur_seen, turn);
    // each warp's first span: the scales may come after K's copy has begun, so its barrier's one arrival is left
    // until they are there
    if (lane < WARPS && turn < cur.n) {
      const int sp = cur.sp0 + turn, row = (sp & 1) * SPAN, at = ids.pid * kv + cur.kvh;
      uint8_t* const k0 = ring + lane * SLOTS * SPAN_BYTES;
      mbar_expect_tx(&sh.full[lane][0], SPAN_BYTES);
      tma_load_3d(k0, tmK, &sh.full[lane][0], 0, row, at);
      mbar_arrive_expect_tx(&sh.full[lane][1], SPAN_BYTES);
      tma_load_3d(k0 + SPAN_BYTES, tmV, &sh.full[lane][1], 0, row, at);
      sh.meta[lane][0] = span_meta(ids, sp);
      mbar_arrive(&sh.full[lane][0]);
      slot = 2;
      use = 1;
      turn += WARPS;
    }
    ids = fetch_ids(cur, cur_table, cur_seen, turn);
  }
  bool ok = true;
  for (int k = 0;; ++k) {
    const int b = k & 1;
    if (k > 0) ok = ok && mbar_wait_uniform(&sh.seg_empty[b], ((k >> 1) & 1) ^ 1, abort_flag, status, STATUS_TIMEOUT_ATTN);
    if (!ok) cur.n = 0;
    if (cur.n && k > 0) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) put_query<F16, NT>(sh, b, r, qw[r], p.scale_log2);
    }
    if (k > 0) publish(b);
    if (!cur.n) break;
    // the next segment's rows and pages are on their way while this one's spans are dealt out
    const Seg next = advance();
    const int* next_table = table;
    const int next_seen = seen;
    const int after = turn + (cur.n > turn ? (cur.n - turn + WARPS - 1) / WARPS * WARPS : 0) - cur.n;  // TURN then
    Ids first = {};
    if (next.n) {
      first = fetch_ids(next, next_table, next_seen, after);
      load_q(next);
    }
    Ids then = fetch_ids(cur, cur_table, cur_seen, turn + WARPS);
    bool left = ok && lane < WARPS && turn < cur.n, v = false;
    uint64_t since = 0;
    while (__any_sync(0xffffffffu, left)) {
      const bool ready = left && mbar_test_wait(&sh.empty[lane][slot], phase ^ 1);
      if (ready) {
        const int sp = cur.sp0 + turn;
        if (!v)
          sh.meta[lane][use & 1] = span_meta(ids, sp);
        mbar_arrive_expect_tx(&sh.full[lane][slot], SPAN_BYTES);
        tma_load_3d(ring + (lane * SLOTS + slot) * SPAN_BYTES, v ? tmV : tmK, &sh.full[lane][slot], 0, (sp & 1) * SPAN,
                    ids.pid * kv + cur.kvh);
        if (++slot == SLOTS) {
          slot = 0;
          phase ^= 1;
        }
        if (v) {
          ++use;
          turn += WARPS;
          left = turn < cur.n;
          ids = then;
          then = fetch_ids(cur, cur_table, cur_seen, turn + WARPS);
        }
        v = !v;
      }
      if (__any_sync(0xffffffffu, ready)) {
        since = 0;
      } else {  // every ring is full
        const uint64_t now = globaltimer();
        if (since == 0) since = now;
        if (__any_sync(0xffffffffu, *abort_flag != 0 || now - since > EXN_WAIT_NS)) {
          if (lane == 0 && !*abort_flag) {
            *abort_flag = 1;
            atomicOr(status, STATUS_TIMEOUT_ATTN);
          }
          __syncwarp();
          left = false;
          ok = false;
        }
        __nanosleep(32);
      }
    }
    turn = after;
    cur = next;
    cur_table = next_table;
    cur_seen = next_seen;
    ids = first;
  }
}

template <bool F16, int NT>
__global__ void __launch_bounds__(AttendCfg<NT>::THREADS, AttendCfg<NT>::CTAS)
    k_cache_attend(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const CacheAttnArgs p, const AttendPlan plan, int* status) {
  using C = AttendCfg<NT>;
  constexpr int ROWS = C::ROWS, WARPS = C::WARPS, SLOTS = C::SLOTS, THREADS = WARPS * 32;  // computing threads
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float (*part_o)[ROWS][128] = reinterpret_cast<float (*)[ROWS][128]>(smem + C::RING);  // [WARPS]
  __shared__ __align__(16) AttendShared<NT> sh;
  volatile int* abort_flag = &sh.abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gi = lane >> 2, ti = lane & 3;
  if (threadIdx.x == 0) {
    sh.abort_word = 0;
    for (int i = 0; i < WARPS * SLOTS; ++i) {
      mbar_init(&sh.full[0][0] + i, 1);
      mbar_init(&sh.empty[0][0] + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.seg_full[i], 1);
      mbar_init(&sh.seg_empty[i], WARPS);
    }
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch();
  if (warp == WARPS) {
    attend_produce<F16, NT>(&tmK, &tmV, p, plan, sh, smem, status);
    return;
  }

  // ---- the computing warps
  auto barrier = [] { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); };
  // the same, and whether all are OK: no warp leaves after a wait that ran out while another waits for it here
  auto together = [](bool ok) -> bool {
    int all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, %2, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(static_cast<int>(ok)), "n"(THREADS)
        : "memory");
    return all != 0;
  };
  const uint32_t ring32 = smem_u32(smem + warp * SLOTS * SPAN_BYTES);
  uint64_t* const full = sh.full[warp];
  uint64_t* const empty = sh.empty[warp];
  int slot = 0;            // of the next tile to read
  uint32_t phase = 0, use = 0;
  int turn = warp;         // spans until this warp's next
  bool ok = true;
  auto step = [&] {
    __syncwarp();  // the tile is read
    if (lane == 0) mbar_arrive(&empty[slot]);
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1;
    }
  };

  for (int k = 0;; ++k) {
    const int b = k & 1;
    ok = together(mbar_wait_uniform(&sh.seg_full[b], (k >> 1) & 1, abort_flag, status, STATUS_TIMEOUT_ATTN));
    if (!ok) break;
    const int n = sh.seg[b].n, nh = sh.seg[b].nh, nrows = sh.seg[b].tok * nh, pos0 = sh.seg[b].pos0;
    if (n == 0) break;
    if (k == 0) {
      const int row0 = sh.seg[0].row0, head0 = sh.seg[0].head0;
      for (int r = warp; r < ROWS; r += WARPS) {
        uint2 w = make_uint2(0u, 0u);
        if (r < nrows)
          w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + (row0 + r / nh) * p.ld_q +
                                                   (head0 + r % nh) * 128 + 4 * lane));
        put_query<F16, NT>(sh, 0, r, w, p.scale_log2);
      }
      barrier();
    }
    // Q^T as the MMA's 32 x 8 operand, hi and lo: this thread's query row is gi (+ 8), its dims 32 ti .. + 31;
    // k-step ks multiplies dims 32 ti + 8 ks .. + 7 (which dims sit where is free as long as q and K agree)
    uint32_t qf[NT][2][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(&sh.q[b][z][nt * 8 + gi][8 * ti + i]);
          qf[nt][z][i] = x.x;
          qf[nt][z][i + 1] = x.y;
          qf[nt][z][i + 2] = x.z;
          qf[nt][z][i + 3] = x.w;
        }
    // the thread's score columns: query rows nt * 8 + 2 ti + {0, 1}
    float qs[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = nt * 8 + 2 * ti + j;
        qs[nt][j] = sh.q_scale[b][row];
        lim[nt][j] = row < nrows ? pos0 + row / nh : -1;
      }

    // a row's maximum and sum of weights; log2 of its sums' unit (a whole number) and of its largest P' so far (top)
    float m[NT][2], l[NT][2], top[NT][2], unit[NT][2], o[NT][8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = top[nt][0] = top[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = unit[nt][0] = unit[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
    }
    for (; turn < n; turn += WARPS) {
      ok = mbar_wait_uniform(&full[slot], phase, abort_flag, status, STATUS_TIMEOUT_ATTN);
      if (!ok) break;
      const float4 meta = sh.meta[warp][use & 1];
      ++use;
      const float skp = meta.x, svp = meta.y;
      const int pos = __float_as_int(meta.z);
      // S^T, 16 positions at a time
      int si[NT][2][2][4];
      {
        const uint32_t at = ring32 + slot * SPAN_BYTES + gi * 128;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // 16 of the thread's 32 dims: chunk 2 ti + half of its rows gi, gi + 8 of 16
          uint4 kc[2][2];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) kc[mt][r] = ld_shared_v4(at + (((2 * ti + half) ^ gi) << 4) + mt * 2048 + r * 1024);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const uint4 x = kc[mt][0], y = kc[mt][1];
                const uint32_t (&q)[8] = qf[nt][z];
                if (half == 0) mma16832_first(si[nt][mt][z], x.x, y.x, x.y, y.y, q[0], q[1]);
                else mma16832(si[nt][mt][z], x.x, y.x, x.y, y.y, q[4], q[5]);
              }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int z = 0; z < 2; ++z)
                mma16832(si[nt][mt][z], kc[mt][0].z, kc[mt][1].z, kc[mt][0].w, kc[mt][1].w, qf[nt][z][4 * half + 2],
                         qf[nt][z][4 * half + 3]);
        }
      }
      step();
      // softmax: one running maximum and sum a query row and warp
      const bool masked = pos + SPAN - 1 > pos0;  // past the last position that every row sees
      const float ev = static_cast<float>((__float_as_int(svp) >> 23) - 127);  // V's scale is 2^ev
      uint32_t pf[NT][2][2];
      float s[NT][2][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float most[2];  // the span's largest scores
        bool need = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float sc = qs[nt][j] * skp, sc_lo = sc * 0x1p-8f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              float& x = s[nt][mt][2 * hh + j];
              x = fmaf(__int_as_float(si[nt][mt][0][2 * hh + j]) - 12582912.f, sc,
                       (__int_as_float(si[nt][mt][1][2 * hh + j]) - 12582912.f) * sc_lo);
              if (masked && pos + mt * 16 + hh * 8 + gi > lim[nt][j]) x = -INFINITY;
            }
          float mx = fmaxf(fmax3(s[nt][0][j], s[nt][0][2 + j], s[nt][1][j]), s[nt][1][2 + j]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          most[j] = mx;
          const float d = mx - m[nt][j];  // infinite where the row sees its first position, NaN where it has seen none
          top[nt][j] = fmaxf(top[nt][j], d + (ev - unit[nt][j]));
          need |= d > 8.f || top[nt][j] > 14.f;
        }
        if (__any_sync(0xffffffffu, need)) {
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float grown = most[j] - m[nt][j], w = 0.f;
            if (grown > 8.f) {
              m[nt][j] = most[j];
              top[nt][j] = grown < INFINITY ? top[nt][j] - grown : ev - unit[nt][j];
            } else {
              grown = 0.f;
            }
            if (top[nt][j] > 14.f || (top[nt][j] < 0.f && m[nt][j] > -INFINITY)) {
              w = fminf(floorf(top[nt][j]), 127.f - unit[nt][j]);
              unit[nt][j] += w;
              top[nt][j] -= w;
            }
            f[j] = fast_exp2(-grown - w);  // at most 2: TOP falls by no more than the maximum grows
            l[nt][j] *= fast_exp2(-grown);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nt][q][j] *= f[j & 1];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float mu = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
          const float to_unit = pow2_of(fminf(fmaxf(ev - unit[nt][j], -127.f), 127.f));
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              float& x = s[nt][mt][2 * hh + j];
              x = fast_exp2(x - mu);
              l[nt][j] += x;
              x *= to_unit;
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            pf[nt][mt][hh] = transpose8x8(pack16<true>(s[nt][mt][2 * hh], s[nt][mt][2 * hh + 1]));
      }
      if (svp != svp) {  // a page of scale NaN: the rows that see a position of it are NaN
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (pos <= lim[nt][j & 1]) o[nt][q][j] = svp;
      }
      ok = mbar_wait_uniform(&full[slot], phase, abort_flag, status, STATUS_TIMEOUT_ATTN);
      if (!ok) break;
      // O^T: dims 16 q + 2 gi, + 1 in the rows gi, gi + 8 of product q; a matrix is 8 positions by 16 codes
      {
        const int row = lane & 15;  // of 16 positions; lanes 16 .. 31 take the next 16 codes of the same rows
        const uint32_t at = ring32 + slot * SPAN_BYTES + row * 128;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t w[4][4];
#pragma unroll
          for (int q = 0; q < 8; q += 2)
            ldmatrix_trans(w[q >> 1], at + mt * 2048 + (((q + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
          for (int q = 0; q < 8; q += 2)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t x = w[q >> 1][2 * z] ^ 0x80808080u, y = w[q >> 1][2 * z + 1] ^ 0x80808080u;
              const uint32_t fr[4] = {v_pair(x, EVEN), v_pair(x, ODD), v_pair(y, EVEN), v_pair(y, ODD)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][q + z], fr, pf[nt][mt][0], pf[nt][mt][1]);
            }
        }
      }
      step();
    }
    turn -= n;

    // ---- join the warps: o = sum_w 2^(m_w - M) o_w, l likewise, in a fixed order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = l[nt][j];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        const int row = nt * 8 + 2 * ti + j;
        const float u = pow2_of(unit[nt][j]);
        if (gi == 0) {
          sh.m[warp][row] = m[nt][j];
          sh.l[warp][row] = t;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<float2*>(&part_o[warp][row][16 * q + 2 * gi]) =
              make_float2(o[nt][q][j] * u, o[nt][q][j + 2] * u);
      }
    const Seg seg = sh.seg[b];
    const int part_len = sh.part_len, lead = sh.lead;
    ok = together(ok);
    if (!ok) break;
    if (lane == 0) mbar_arrive(&sh.seg_empty[b]);
    const bool whole = n == seg.spans;
    // a row's four values at 4 (x & 31), normalised and stored
    auto store = [&](int row, int x, float4 a, float t) {
      const float inv = t == 0.f ? 0.f : 1.f / t;  // a row that sees no position is 0
      const int tok = row / nh, hd = row - tok * nh;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (seg.row0 + tok) * p.ld_out + (seg.head0 + hd) * 128 +
                                (x & 31) * 4) = make_uint2(pack16<F16>(a.x * inv, a.y * inv), pack16<F16>(a.z * inv, a.w * inv));
    };
    const int mine = 2 * blockIdx.x + (seg.sp0 ? 0 : 1);
    for (int x = threadIdx.x; x < nrows * 32; x += THREADS) {
      const int row = x >> 5;
      float mx = sh.m[0][row];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, sh.m[w][row]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float t = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float c = fast_exp2(sh.m[w][row] - mu);
        const float4 y = reinterpret_cast<const float4*>(part_o[w][row])[x & 31];
        t += c * sh.l[w][row];
        a.x += c * y.x;
        a.y += c * y.y;
        a.z += c * y.z;
        a.w += c * y.w;
      }
      if (whole) {
        store(row, x, a, t);
      } else {
        float* dst = plan.part + (static_cast<long long>(mine) * ROWS + row) * 132;
        *reinterpret_cast<float4*>(dst + (x & 31) * 4) = a;
        if ((x & 31) == 0) *reinterpret_cast<float2*>(dst + 128) = make_float2(mx, t);
      }
    }
    barrier();  // the join's memory is free, the part is written
    if (whole) continue;

    // ---- an item that several CTAs share: the last one to get here joins its parts
    const unsigned first = seg.item + lead;
    const int c0 = static_cast<int>(first / static_cast<unsigned>(part_len));
    const int parts = static_cast<int>((first + seg.spans - 1) / static_cast<unsigned>(part_len)) - c0 + 1;
    auto part_of = [&](int i) { return i == 0 ? 2 * c0 + 1 : 2 * (c0 + i); };
    if (threadIdx.x == 0) {
      fence_acq_rel();  // after this part's stores (the block's, by the barrier above)
      sh.taken = count_part(plan.count + c0, plan.tag) + 1 == parts;
      if (sh.taken) {
        fence_acq_rel();  // the others' parts are read after their counts
        plan.count[c0] = 0;
      }
    }
    barrier();
    if (sh.taken) {
      // a row's four values at 4 (x & 31) of eight parts, on their way before they are needed
      const auto fetch = [&](int x, int i0, float4 (&y)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (x < nrows * 32 && i0 + i < parts)
            y[i] = __ldcg(reinterpret_cast<const float4*>(
                              plan.part + (static_cast<long long>(part_of(i0 + i)) * ROWS + (x >> 5)) * 132) + (x & 31));
      };
      int x = threadIdx.x, i0 = 0;
      float4 y[8], a = make_float4(0.f, 0.f, 0.f, 0.f);
      fetch(x, i0, y);
      // each part's weight 2^(m - M) and each row's sum (in the join's memory), GROUP threads a row
      constexpr int GROUP = THREADS / ROWS >= 16 ? 16 : 8;
      static_assert(GROUP * ROWS <= THREADS && GROUP * ROWS % 32 == 0, "whole warps");
      float* weight = &part_o[0][0][0];
      float* part_sum = weight + plan.ctas * ROWS;  // an item has at most CTAS parts: room for both (attend_plan)
      if (threadIdx.x < GROUP * ROWS) {
        const int row = threadIdx.x / GROUP, sub = threadIdx.x % GROUP;
        float mx = -INFINITY, t = 0.f;
        if (row < nrows)
          for (int i = sub; i < parts; i += GROUP) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(
                plan.part + (static_cast<long long>(part_of(i)) * ROWS + row) * 132 + 128));
            weight[i * ROWS + row] = ml.x;
            part_sum[i * ROWS + row] = ml.y;
            mx = fmaxf(mx, ml.x);
          }
#pragma unroll
        for (int x = GROUP / 2; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float mu = mx == -INFINITY ? 0.f : mx;
        if (row < nrows)
          for (int i = sub; i < parts; i += GROUP) {
            const float c = fast_exp2(weight[i * ROWS + row] - mu);
            weight[i * ROWS + row] = c;
            t += c * part_sum[i * ROWS + row];
          }
#pragma unroll
        for (int x = GROUP / 2; x > 0; x >>= 1) t += __shfl_xor_sync(0xffffffffu, t, x);
        if (sub == 0) sh.l[0][row] = t;
      }
      barrier();
      while (x < nrows * 32) {
        const int row = x >> 5, next_i = i0 + 8 < parts ? i0 + 8 : 0, next_x = next_i ? x : x + THREADS;
        float4 z[8];
        fetch(next_x, next_i, z);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < parts) {
            const float c = weight[(i0 + i) * ROWS + row];
            a.x += c * y[i].x;
            a.y += c * y[i].y;
            a.z += c * y[i].z;
            a.w += c * y[i].w;
          }
        if (next_i == 0) {
          store(row, x, a, sh.l[0][row]);
          a = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = z[i];
        x = next_x;
        i0 = next_i;
      }
      barrier();  // the join's memory is free again
    }
  }
  if (!ok) {  // the copies in flight to this warp's ring land before the CTA leaves
    volatile int no_abort = 0;
    for (int i = 0; i < SLOTS; ++i) mbar_wait(&full[i], phase ^ (i < slot ? 1u : 0u), &no_abort, nullptr, 0, 100000000ull);
  }
}

// A bit that a kernel on another stream sets meanwhile is in what is taken or in what is left
__global__ void k_status_take(int* status) { status[1] = atomicExch(status, 0); }

// A number that no other launch of this process has and that is no likely memory content
unsigned long long launch_tag() {
  static std::atomic<unsigned long long> next{
      static_cast<unsigned long long>(std::chrono::system_clock::now().time_since_epoch().count()) * 0x9e3779b97f4a7c15ull};
  unsigned long long t;
  do t = next.fetch_add(0x9e3779b97f4a7c15ull) << 16;  // an odd step: every 48-bit number once
  while (t == 0);                                      // 0: no launch's
  return t;
}

}  // namespace

int cache_write_launch(const CacheArgs& c, int f16, const int* offsets, long long rows, const void* k, long long ld_k,
                       const void* v, long long ld_v, int* d_status, cudaStream_t st) {
  const long long blocks = (rows / kPage + 2ll * c.nseq) * c.kv_heads * 2;
  if (blocks > 0x7fffffffll) return -1;
  return static_cast<int>(launch_pdl(f16 ? k_cache_write<true> : k_cache_write<false>,
                                     dim3(static_cast<unsigned>(blocks)), dim3(128), 0, st, c, offsets, rows,
                                     static_cast<const uint16_t*>(k), ld_k, static_cast<const uint16_t*>(v), ld_v, d_status));
}

int cache_read_launch(const CacheArgs& c, int f16, const int* offsets, long long rows, void* k, long long ld_k,
                      void* v, long long ld_v, int* d_status, cudaStream_t st) {
  const long long blocks = (rows / kPage + 2ll * c.nseq) * c.kv_heads * 2;
  if (blocks > 0x7fffffffll) return -1;
  return static_cast<int>(launch_pdl(f16 ? k_cache_read<true, false> : k_cache_read<false, false>,
                                     dim3(static_cast<unsigned>(blocks)), dim3(128), 0, st, c, offsets, rows,
                                     static_cast<uint16_t*>(k), ld_k, static_cast<uint16_t*>(v), ld_v, d_status));
}

static long long dense_blocks(const CacheArgs& c) { return static_cast<long long>(c.nseq) * c.table_ld * c.kv_heads * 2; }
static int dense_launch(const CacheArgs& c, int f16, void* k, void* v, int* d_status, cudaStream_t st) {
  const long long ld = static_cast<long long>(c.kv_heads) * 128;
  return static_cast<int>(launch_pdl(f16 ? k_cache_read<true, true> : k_cache_read<false, true>,
                                     dim3(static_cast<unsigned>(dense_blocks(c))), dim3(128), 0, st, c,
                                     static_cast<const int*>(nullptr), 0ll, static_cast<uint16_t*>(k), ld,
                                     static_cast<uint16_t*>(v), ld, d_status));
}

int status_take_launch(int* status, cudaStream_t st) {
  void* args[] = {&status};
  return static_cast<int>(cudaLaunchKernel(reinterpret_cast<const void*>(k_status_take), dim3(1), dim3(1), args, 0, st));
}

int cache_prepare() {
  cudaError_t e = cudaSuccess;
  for (auto* k : {k_cache_attend<false, 1>, k_cache_attend<true, 1>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, AttendCfg<1>::SMEM);
  for (auto* k : {k_cache_attend<false, 2>, k_cache_attend<true, 2>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, AttendCfg<2>::SMEM);
  return static_cast<int>(e);
}

// Few rows (tokens times the query heads of a key/value head) read the codes directly, 16 at a time; with
// more, the cache is turned into 16 bits once and read by the packed kernel's tensor-core tiles.  us either
// way, codes / 16 bits (32 heads over 8):
//   rows a sequence              32          64          96         128         192
//   1 sequence of 8000       23 / 37     31 / 37     32 / 37     42 / 37     54 / 40
//   8 sequences of 2000      24 / 44     47 / 50     62 / 50     76 / 51    105 / 53
//   32 sequences of 4000    130 / 245   236 / 246   339 / 248   443 / 252   657 / 269
// so the bound is 64 rows a sequence and 64 more for the launch.  Tables with room for more positions than one
// launch can turn into 16 bits leave the codes.
static long long dense_rows(const CacheArgs& c) { return static_cast<long long>(c.nseq) * c.table_ld * kPage; }
static bool dense_path(const CacheArgs& c, int heads, long long rows) {
  return rows * (heads / c.kv_heads) > 64 * (c.nseq + 1ll) && dense_rows(c) <= 0x7fffffffll && dense_blocks(c) <= 0x7fffffffll;
}

// the cut of the direct path's work: a wave of CTAs, tiles of 8 or 16 query rows.  us with tiles of 8 / 16
// (bf16; the codes are read again for every tile):
//   rows a sequence                            4             8            12            32
//   1 sequence of 64000, 32 heads over 8   34 / 41       38 / 43       49 / 43       80 / 68
//   8 of 8000, 32 over 8                   32 / 40       33 / 41       50 / 42       92 / 69
//   64 of 4000, 32 over 8                  96 / 123      97 / 126     175 / 129     334 / 235
// so 16 when the sequences' rows (on average) need more than 8.
static AttendPlan attend_plan(const CacheArgs& c, int heads, long long rows, int sms, void* ws) {
  AttendPlan p;
  const int g = heads / c.kv_heads;
  const long long per = (rows + c.nseq - 1) / c.nseq;  // new tokens a sequence
  const int nt = per * g > 8 ? 2 : 1;
  p.nt = nt;
  p.hpt = g < 8 * nt ? g : 8 * nt;
  p.head_tiles = (g + p.hpt - 1) / p.hpt;
  const int room = 8 * nt / p.hpt;
  p.tpt = per < room ? static_cast<int>(per) : room;
  // a wave, but no more CTAs than the join's memory has room for an item's parts (two floats a row and part)
  const int wave = sms * (nt == 1 ? AttendCfg<1>::CTAS : AttendCfg<2>::CTAS);
  const int room_for = (nt == 1 ? AttendCfg<1>::JOIN : AttendCfg<2>::JOIN) / (8 * nt * 8);
  p.ctas = wave < room_for ? wave : room_for;
  p.tag = 0;
  p.part = static_cast<float*>(ws);
  p.count = reinterpret_cast<unsigned long long*>(p.part + 2ll * p.ctas * 8 * nt * 132);
  return p;
}
// enough for ROWS and for any fewer
size_t cache_attention_workspace(const CacheArgs& c, int heads, long long rows, int sms) {
  static_assert(AttendCfg<1>::CTAS >= AttendCfg<2>::CTAS, "the most CTAs, parts of the most rows");
  const size_t codes = static_cast<size_t>(sms) * AttendCfg<1>::CTAS * (2 * AttendCfg<2>::ROWS * 132 * 4 + 8);
  const size_t dense = static_cast<size_t>(dense_rows(c)) * c.kv_heads * 128 * 2 * 2;
  return dense_path(c, heads, rows) && dense > codes ? dense : codes;
}

static int attend_launch(const CacheAttnArgs& a, void* ws, int sms, int* d_status, cudaStream_t st) {
  AttendPlan p = attend_plan(a.c, a.heads, a.rows, sms, ws);
  p.tag = launch_tag();
  const bool one = p.nt == 1;
  CUtensorMap tk, tv;
  const uint64_t d[3] = {128, kPage, static_cast<uint64_t>(a.c.pages) * a.c.kv_heads};
  const uint64_t s[2] = {128, PAGE_BYTES};
  const uint32_t b[3] = {128, SPAN, 1};
  if (make_tmap(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.c.k, 3, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B) ||
      make_tmap(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.c.v, 3, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B))
    return -4;
  const int threads = one ? AttendCfg<1>::THREADS : AttendCfg<2>::THREADS, smem = one ? AttendCfg<1>::SMEM : AttendCfg<2>::SMEM;
  return static_cast<int>(launch_pdl(one ? (a.f16 ? k_cache_attend<true, 1> : k_cache_attend<false, 1>)
                                         : (a.f16 ? k_cache_attend<true, 2> : k_cache_attend<false, 2>),
                                     dim3(p.ctas), dim3(threads), smem, st, tk, tv, a, p, d_status));
}

int cache_attention(const CacheAttnArgs& a, void* ws, size_t ws_bytes, int sms, const int (&fit)[3], int* d_status,
                    cudaStream_t st) {
  const CacheArgs& c = a.c;
  if (ws_bytes < cache_attention_workspace(c, a.heads, a.rows, sms)) return -1;
  if (!dense_path(c, a.heads, a.rows)) return attend_launch(a, ws, sms, d_status, st);
  uint16_t* k = static_cast<uint16_t*>(ws);
  uint16_t* v = k + static_cast<size_t>(dense_rows(c)) * c.kv_heads * 128;
  const int r = dense_launch(c, a.f16, k, v, d_status, st);
  if (r) return r;
  PackedArgs p;
  p.f16 = a.f16;
  p.heads = a.heads;
  p.kv_heads = c.kv_heads;
  p.nseq = c.nseq;
  p.q_offsets = a.offsets;
  p.kv_lens = c.lens;
  p.kv_stride = static_cast<long long>(c.table_ld) * kPage;
  p.rows = a.rows;
  p.kv_rows = dense_rows(c);
  p.q = a.q;
  p.k = k;
  p.v = v;
  p.out = a.out;
  p.ld_q = a.ld_q;
  p.ld_k = p.ld_v = static_cast<long long>(c.kv_heads) * 128;
  p.ld_out = a.ld_out;
  p.scale_log2 = a.scale_log2;
  for (int i = 0; i < 3; ++i) p.fit[i] = fit[i];
  return packed_launch(p, d_status, st);
}

}  // namespace exn
