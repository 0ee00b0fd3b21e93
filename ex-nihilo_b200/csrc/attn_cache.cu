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

__device__ __forceinline__ int to_code(float x, float top) { return __float2int_rn(fminf(fmaxf(x, -top), top)); }

// The sequence whose page slots hold SLOT: s owns the slots from floor(start_s / 64) + 2 s on, of which
// its rows, consecutive positions, touch at most ceil(count / 64) + 1 pages.  All threads; -1: none.
__device__ __forceinline__ int find_sequence(const int* offsets, const int* lens, int nseq, long long rows, int slot,
                                             int* found, int* status) {
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < nseq; s += blockDim.x) {
    const long long a = offsets[s], b = offsets[s + 1];
    if (a < 0 || b < a || b > rows || lens[s] < b - a) {
      if (blockIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      continue;
    }
    if (b == a) continue;
    const long long first = a / kPage + 2ll * s;
    const long long p0 = (lens[s] - (b - a)) / kPage, p1 = (lens[s] - 1) / kPage;
    if (slot >= first && slot <= first + p1 - p0) *found = s;
  }
  __syncthreads();
  return *found;
}

// ---- write: one block = one page touched by the call's rows, one key/value head; threads 0..127 take
// K, 128..255 V, eight threads a row of 128 values.  Bound by the bytes: 2 in and 1 out a value.
template <bool F16>
__global__ void __launch_bounds__(256) k_cache_write(const CacheArgs c, const int* __restrict__ offsets,
                                                     long long rows, const uint16_t* __restrict__ k, long long ld_k,
                                                     const uint16_t* __restrict__ v, long long ld_v, int* status) {
  __shared__ int found;
  __shared__ float red[8];
  const int slot = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  griddep_wait();
  griddep_launch();
  const int s = find_sequence(offsets, c.lens, c.nseq, rows, slot, &found, status);
  if (s < 0) return;
  const int start = offsets[s], count = offsets[s + 1] - start;
  const int pos0 = c.lens[s] - count;
  const int page_i = pos0 / kPage + slot - (start / kPage + 2 * s);
  const int page = page_i < c.table_ld ? c.table[static_cast<long long>(s) * c.table_ld + page_i] : -1;
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    return;
  }
  const int lo = max(pos0, page_i * kPage) - page_i * kPage;             // rows of the page written: lo .. hi - 1
  const int hi = min(pos0 + count, (page_i + 1) * kPage) - page_i * kPage;
  const long long row0 = start + static_cast<long long>(page_i) * kPage - pos0;  // the row of the page's position 0
  const bool is_v = threadIdx.x >= 128;
  const int tid = threadIdx.x & 127, sub = tid & 7, r0 = tid >> 3;  // 16 values at 16 sub of rows r0, r0 + 16, ..
  const uint16_t* src = (is_v ? v : k) + h * 128 + sub * 16;
  const long long ld = is_v ? ld_v : ld_k;
  const long long head = static_cast<long long>(page) * c.kv_heads + h;
  int8_t* dst = (is_v ? c.v : c.k) + head * PAGE_BYTES + sub * 16;
  float* scale = (is_v ? c.v_scale : c.k_scale) + head;

  uint4 x[4][2];
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (r >= lo && r < hi) {
      const uint4* p = reinterpret_cast<const uint4*>(src + (row0 + r) * ld);
      x[i][0] = __ldg(p);
      x[i][1] = __ldg(p + 1);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = unpack16<F16>(reinterpret_cast<const uint32_t*>(&x[i][0])[j]);
      amax = fmax3(amax, fabsf(f.x), fabsf(f.y));
      bad |= !(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY);
    }
  if (bad) amax = INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const float before = lo > 0 ? *scale : 0.f;  // what the page holds already (none when it starts anew)
  __syncthreads();
  const int w0 = is_v ? 4 : 0;
  amax = fmaxf(fmaxf(red[w0], red[w0 + 1]), fmaxf(red[w0 + 2], red[w0 + 3]));
  const bool poisoned = !(amax < INFINITY) || before != before;
  const float mine = pow2(scale_exponent(poisoned ? 0.f : amax));
  const float now = fmaxf(mine, before);
  const float inv = 1.f / now;  // exact: a power of two between 2^-122 and 2^126
  const float top = now < 0x1p122f ? 127.f : 63.f;  // 64 * 2^122 would be infinite
  if (lo > 0 && !poisoned && now > before) {  // the codes that are there, in the larger unit
    const float f = before * inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 16 * i;
      if (r < lo) {
        uint4* p = reinterpret_cast<uint4*>(dst + r * 128);
        uint4 w = *p;
        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
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
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i;
    if (r >= lo && r < hi) {
      uint4 w;
      uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = unpack16<F16>(reinterpret_cast<const uint32_t*>(&x[i][0])[2 * j]);
        const float2 b = unpack16<F16>(reinterpret_cast<const uint32_t*>(&x[i][0])[2 * j + 1]);
        const float f[4] = {a.x, a.y, b.x, b.y};
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          n |= (static_cast<uint32_t>(poisoned ? 0 : to_code(f[e] * inv, top)) & 0xffu) << (8 * e);
        u[j] = n;
      }
      *reinterpret_cast<uint4*>(dst + r * 128) = w;
    }
  }
  if (tid == 0) *scale = poisoned ? __uint_as_float(0x7fffffffu) : now;
}

// ---- read: the same blocks; code * scale in 16 bits (exact in bf16; rounded once where fp16's range
// ends).  DENSE: every position, to row s * table_ld * 64 + position.  Bound by the bytes: 1 in, 2 out.
template <bool F16, bool DENSE>
__global__ void __launch_bounds__(256) k_cache_read(const CacheArgs c, const int* __restrict__ offsets,
                                                    long long rows, uint16_t* __restrict__ k, long long ld_k,
                                                    uint16_t* __restrict__ v, long long ld_v, int* status) {
  __shared__ int found;
  const int slot = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  griddep_wait();
  griddep_launch();
  int s, page_i, lo, hi;
  long long row0;
  if (DENSE) {
    s = slot / c.table_ld;
    page_i = slot - s * c.table_ld;
    const int len = c.lens[s];
    if (len < 0 || len > static_cast<long long>(c.table_ld) * kPage) {
      if (page_i == 0 && threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      return;
    }
    if (len <= page_i * kPage) return;
    lo = 0;  // the last page whole: the rows behind the sequence's last are then finite, as its codes are
    hi = kPage;
    row0 = static_cast<long long>(slot) * kPage;
  } else {
    s = find_sequence(offsets, c.lens, c.nseq, rows, slot, &found, status);
    if (s < 0) return;
    const int start = offsets[s], count = offsets[s + 1] - start;
    const int pos0 = c.lens[s] - count;
    page_i = pos0 / kPage + slot - (start / kPage + 2 * s);
    lo = max(pos0, page_i * kPage) - page_i * kPage;
    hi = min(pos0 + count, (page_i + 1) * kPage) - page_i * kPage;
    row0 = start + static_cast<long long>(page_i) * kPage - pos0;
  }
  const int page = page_i < c.table_ld ? c.table[static_cast<long long>(s) * c.table_ld + page_i] : -1;
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    return;
  }
  const bool is_v = threadIdx.x >= 128;
  const int tid = threadIdx.x & 127, sub = tid & 7, r0 = tid >> 3;
  const long long head = static_cast<long long>(page) * c.kv_heads + h;
  const int8_t* src = (is_v ? c.v : c.k) + head * PAGE_BYTES + sub * 16;
  const float scale = (is_v ? c.v_scale : c.k_scale)[head];
  uint16_t* dst = (is_v ? v : k) + h * 128 + sub * 16;
  const long long ld = is_v ? ld_v : ld_k;
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i;
    if (r >= lo && r < hi) w[i] = *reinterpret_cast<const uint4*>(src + r * 128);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i;
    if (r < lo || r >= hi) continue;
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[i]);
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t pair = u[j >> 1] >> (16 * (j & 1));
      o[j] = pack16<F16>(static_cast<float>(static_cast<int8_t>(pair)) * scale,
                         static_cast<float>(static_cast<int8_t>(pair >> 8)) * scale);
    }
    uint4* p = reinterpret_cast<uint4*>(dst + (row0 + r) * ld);
    p[0] = make_uint4(o[0], o[1], o[2], o[3]);
    p[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// ---- attention of a few rows over the codes
//
// One cluster = one tile of up to 8 NT query rows (tokens times the query heads that read one
// key/value head) of a sequence; its WARPS * CTAs warps take the sequence's pages in turn, each with
// its own running maximum, sum and output, joined at the end through shared memory and the cluster's.
// Bound by the codes' bytes (a code takes part in 4 g c operations), as long as the conversions to
// 16 bits keep up: they are the bulk of the instructions, so
//   * both products run on fp16 MMAs (m16n8k16), whichever type q has: an int8 code becomes fp16
//     exactly with one byte permute and one subtraction a pair (1024 + (code + 128) is fp16 0x6400 |
//     byte); a row of q is scaled by a power of two to lie below 2^15 (bf16's 8 bits fit fp16's 11;
//     what is 2^-29 of the row's largest is lost), P is at most 1;
//   * codes are the 16-row operand and the queries the 8 columns: S^T = K Q^T, O^T = V^T P^T, so 8
//     rows of queries waste nothing; P^T turns from the first product's layout to the second's with
//     movmatrix;
//   * the scales stay out of the products: 2^ek multiplies the scores, 2^ev the page's fp32 sums.
// Each warp streams its pages with TMA through a ring of its own (K_0 V_0 K_1 ..., 8 KB each, 128-byte
// swizzle: the 16-byte reads below touch every bank once) and re-fills a slot as soon as it has
// read it.
constexpr int MAX_CLUSTER = 16;

template <int WARPS, int NT>
struct AttendCfg {
  static constexpr int SLOTS = 3;
  static constexpr int RING = WARPS * SLOTS * PAGE_BYTES;
  static constexpr int ROWS = 8 * NT;
  static constexpr int OFF_BAR = RING;
  static constexpr int OFF_JOIN = OFF_BAR + WARPS * SLOTS * 8 + 64;  // the CTA's joined m, l [ROWS] each
  static constexpr int SMEM = OFF_JOIN + 2 * ROWS * 4 + 1024;
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
// two pairs of biased codes (code + 128) to fp16: bytes 0, 1 and bytes 2, 3
__device__ __forceinline__ uint32_t codes_lo(uint32_t u) {
  const uint32_t h = __byte_perm(u, 0x64646464u, 0x4140);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t u) {
  const uint32_t h = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

template <bool F16, int WARPS, int NT>
__global__ void __launch_bounds__(WARPS * 32)
    k_cache_attend(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const CacheAttnArgs p, int hpt, int head_tiles, int tpt, int* status) {
  using C = AttendCfg<WARPS, NT>;
  constexpr int ROWS = C::ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  int* flags = reinterpret_cast<int*>(smem + C::OFF_BAR + WARPS * C::SLOTS * 8);  // found, abort
  float* join_m = reinterpret_cast<float*>(smem + C::OFF_JOIN);
  float* join_l = join_m + ROWS;
  volatile int* abort_flag = flags + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gi = lane >> 2, ti = lane & 3;
  const int ncta = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int kv = p.c.kv_heads, g = p.heads / kv;
  int item = blockIdx.x / ncta;
  const int kvh = item % kv;
  item /= kv;
  const int ht = item % head_tiles, slot = item / head_tiles;
  if (threadIdx.x == 0) {
    flags[0] = -1;
    flags[1] = 0;
    for (int i = 0; i < WARPS * C::SLOTS; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  griddep_wait();
  griddep_launch();
  __syncthreads();
  // sequence s owns the row tiles from floor(start_s / tpt) + s on (from start_s when tpt is 1)
  for (int s = threadIdx.x; s < p.c.nseq; s += WARPS * 32) {
    const long long a = p.offsets[s], b = p.offsets[s + 1];
    if (a < 0 || b < a || b > p.rows || p.c.lens[s] < 0) {
      if (blockIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
      continue;
    }
    const long long first = tpt == 1 ? a : a / tpt + s;
    if (slot >= first && slot < first + (b - a + tpt - 1) / tpt) flags[0] = s;
  }
  __syncthreads();
  const int seq = flags[0];
  if (seq < 0) return;  // the whole cluster: every CTA of it has the same slot
  const int start = p.offsets[seq], count = p.offsets[seq + 1] - start;
  const int t0 = (slot - (tpt == 1 ? start : start / tpt + seq)) * tpt;  // first token of the tile
  const int ntok = min(tpt, count - t0);
  const int delta = p.c.lens[seq] - count;                               // token t is position t + delta
  const int h0 = ht * hpt, nh = min(hpt, g - h0);                        // its heads kvh g + h0 ..
  const int nrows = ntok * nh;
  const int seen = t0 + ntok + delta;  // positions the tile's last row sees
  int npages = seen > 0 ? (seen + kPage - 1) / kPage : 0;
  if (npages > p.c.table_ld) {
    if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_ARG);
    npages = p.c.table_ld;
  }
  const int* table = p.c.table + static_cast<long long>(seq) * p.c.table_ld;
  const int w0 = rank * WARPS + warp, wn = ncta * WARPS;
  const int mine = npages > w0 ? (npages - w0 + wn - 1) / wn : 0;  // pages w0, w0 + wn, ..

  // Q^T as the MMA's 16 x 8 operand: this thread's query row is gi (+ 8), its dims 32 ti .. + 31;
  // k-step ks multiplies dims 32 ti + 4 ks .. + 3.  The row's exponent is brought below 2^15.
  uint32_t qf[NT][16];
  int qexp[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = nt * 8 + gi;
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < nrows) {
      const int tok = row / nh, hd = row - tok * nh;
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) +
                                                        (start + t0 + tok) * p.ld_q + (kvh * g + h0 + hd) * 128 + 32 * ti);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldg(src + i);
    }
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if (F16) {
      qexp[nt] = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) qf[nt][i] = u[i];
    } else {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = unpack16<false>(u[i]);
        mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127;  // floor(log2 mx)
      qexp[nt] = mx > 0.f && e < 128 ? max(e - 14, -112) : 0;           // 0 as well for an infinity
      const float f0 = pow2(-qexp[nt]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = unpack16<false>(u[i]);
        qf[nt][i] = pack16<true>(f.x * f0, f.y * f0);
      }
    }
  }
  // the thread's score columns: query rows nt * 8 + 2 ti + {0, 1}
  float qs[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = nt * 8 + 2 * ti + j;
      qs[nt][j] = p.scale_log2 * pow2(__shfl_sync(0xffffffffu, qexp[nt], (2 * ti + j) * 4));
      lim[nt][j] = row < nrows ? t0 + row / nh + delta : -1;
    }

  // ---- the pages, one at a time; lane 0 keeps up to SLOTS tiles ahead in flight
  uint8_t* ring = smem + warp * C::SLOTS * PAGE_BYTES;
  uint64_t* bar = full + warp * C::SLOTS;
  const uint32_t ring32 = smem_u32(ring);
  float m[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
  }
  // page ids and scales of the warp's next 32 pages, one a lane
  int pid = 0;
  float sk = 0.f, sv = 0.f;
  auto fetch_ids = [&](int i0) {
    const int i = i0 + lane;
    pid = 0;
    sk = sv = 0.f;
    if (i < mine) {
      pid = __ldg(table + w0 + i * wn);
      if (pid < 0 || pid >= p.c.pages) {  // not a page: its positions are left out (a scale is never negative)
        atomicOr(status, STATUS_BAD_ARG);
        pid = 0;
        sk = -1.f;
      } else {
        sk = __ldg(p.c.k_scale + static_cast<long long>(pid) * kv + kvh);
        sv = __ldg(p.c.v_scale + static_cast<long long>(pid) * kv + kvh);
      }
    }
  };
  // tile t of the warp: K of its page t / 2 for even t, V for odd t
  auto issue = [&](int t, int page) {
    const int sl = t % C::SLOTS;
    mbar_arrive_expect_tx(&bar[sl], PAGE_BYTES);
    tma_load_3d(ring + sl * PAGE_BYTES, (t & 1) ? &tmV : &tmK, &bar[sl], 0, 0, page * kv + kvh);
  };
  int issued = 0;
  if (mine > 0) {
    fetch_ids(0);
    const int p0 = __shfl_sync(0xffffffffu, pid, 0), p1 = __shfl_sync(0xffffffffu, pid, 1);
    if (lane == 0) {
      issue(0, p0);
      issue(1, p0);
      if (mine > 1) issue(2, p1);
    }
    issued = mine > 1 ? 3 : 2;
  }
  int next_pid = 0;  // page i + 1's id, across a change of the 32 in the lanes
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const float skp = __shfl_sync(0xffffffffu, sk, i & 31), svp = __shfl_sync(0xffffffffu, sv, i & 31);
    const int page_pos = skp < 0.f ? 0x7ffffff0 - kPage : (w0 + i * wn) * kPage;
    if ((i & 31) == 31 && i + 1 < mine) fetch_ids(i + 1);
    next_pid = __shfl_sync(0xffffffffu, pid, (i + 1) & 31);
    ok = ok && mbar_wait_uniform(&bar[(2 * i) % C::SLOTS], static_cast<uint32_t>((2 * i) / C::SLOTS) & 1, abort_flag, status,
                                 STATUS_TIMEOUT_ATTN);
    if (!ok) break;
    // S^T, 16 positions at a time
    float s[NT][4][4];
    {
      const uint32_t base = ring32 + (2 * i) % C::SLOTS * PAGE_BYTES;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nt][mt][j] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // 16 of the thread's 32 dims: chunk 2 ti + half of its rows
          uint32_t a[4], b[4];
          const uint32_t off = static_cast<uint32_t>((((2 * ti + half) ^ gi) << 4) + (mt * 16 + gi) * 128);
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(base + off) : "memory");
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(base + off + 1024) : "memory");
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint32_t ua = a[ks] ^ 0x80808080u, ub = b[ks] ^ 0x80808080u;
            const uint32_t fr[4] = {codes_lo(ua), codes_lo(ub), codes_hi(ua), codes_hi(ub)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(s[nt][mt], fr, qf[nt][2 * (half * 4 + ks)], qf[nt][2 * (half * 4 + ks) + 1]);
          }
        }
      }
    }
    // K's slot is free (its reads fed the products above): page i + 1's V, or the K after
    __syncwarp();
    if (issued < 2 * mine) {
      // tile 2 i + 3 = V of page i + 1
      if (lane == 0) issue(2 * i + 3, next_pid);
      ++issued;
    }
    // softmax: one running maximum and sum a query row and warp
    float corr[NT][2];
    uint32_t pf[NT][4][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float f = qs[nt][j] * skp;
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float& x = s[nt][mt][2 * hh + j];
            x = page_pos + mt * 16 + hh * 8 + gi > lim[nt][j] ? -INFINITY : x * f;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][j], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        corr[nt][j] = fast_exp2(m[nt][j] - mu);
        m[nt][j] = mn;
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float& x = s[nt][mt][2 * hh + j];
            x = fast_exp2(x - mu);
            sum += x;
          }
        l[nt][j] = l[nt][j] * corr[nt][j] + sum;
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
          pf[nt][mt][hh] = transpose8x8(pack16<true>(s[nt][mt][2 * hh], s[nt][mt][2 * hh + 1]));
    }
    ok = mbar_wait_uniform(&bar[(2 * i + 1) % C::SLOTS], static_cast<uint32_t>((2 * i + 1) / C::SLOTS) & 1, abort_flag,
                           status, STATUS_TIMEOUT_ATTN);
    if (!ok) break;
    // O^T: dims 16 gi + 2 i, + 1 in the rows gi, gi + 8 of product i
    float acc[NT][8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nt][q][j] = 0.f;
    {
      const uint32_t base = ring32 + (2 * i + 1) % C::SLOTS * PAGE_BYTES;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        uint32_t w[4][4];  // positions 2 ti, 2 ti + 1, 2 ti + 8, 2 ti + 9 of the 16, dims 16 gi .. + 15
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 2 * ti + (r & 1) + (r >> 1) * 8;
          const uint32_t off = static_cast<uint32_t>(((gi ^ (row & 7)) << 4) + (mt * 16 + row) * 128);
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w[r][0]), "=r"(w[r][1]), "=r"(w[r][2]), "=r"(w[r][3])
                       : "r"(base + off)
                       : "memory");
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t sel = (q & 1) ? 0x7362 : 0x5140;
          const uint32_t x = __byte_perm(w[0][q >> 1], w[1][q >> 1], sel) ^ 0x80808080u;
          const uint32_t y = __byte_perm(w[2][q >> 1], w[3][q >> 1], sel) ^ 0x80808080u;
          const uint32_t fr[4] = {codes_lo(x), codes_hi(x), codes_lo(y), codes_hi(y)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][q], fr, pf[nt][mt][0], pf[nt][mt][1]);
        }
      }
    }
    __syncwarp();
    if (issued < 2 * mine) {  // V's slot is free: tile 2 i + 4 = K of page i + 2
      const int np = __shfl_sync(0xffffffffu, pid, (i + 2) & 31);
      int id = np;
      if (((i + 2) & 31) == 0) id = __ldg(table + w0 + (i + 2) * wn);  // the lanes still hold the 32 before
      if (id < 0 || id >= p.c.pages) id = 0;
      if (lane == 0) issue(2 * i + 4, id);
      ++issued;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // a page that the row does not see at all adds nothing, whatever its scale
      const float sv0 = page_pos > lim[nt][0] ? 0.f : svp, sv1 = page_pos > lim[nt][1] ? 0.f : svp;
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[nt][q][j] = o[nt][q][j] * corr[nt][j & 1] + ((j & 1) ? sv1 : sv0) * acc[nt][q][j];
    }
  }
  if (!ok && lane == 0) {  // the copies in flight land before the ring is used again
    volatile int no_abort = 0;
    for (int t = issued - C::SLOTS < 0 ? 0 : issued - C::SLOTS; t < issued; ++t)
      mbar_wait(&bar[t % C::SLOTS], static_cast<uint32_t>(t / C::SLOTS) & 1, &no_abort, nullptr, 0);
  }

  // ---- join: the warps' parts through shared memory (over the ring), then the CTAs' through the
  // cluster's.  o = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w in a fixed order.
  __syncthreads();
  float* part_o = reinterpret_cast<float*>(smem);                                // [WARPS][ROWS][128]
  float* part_m = part_o + WARPS * ROWS * 128;                                   // [WARPS][ROWS]
  float* part_l = part_m + WARPS * ROWS;
  float* cta_o = part_l + WARPS * ROWS;                                          // [ROWS][128]
  static_assert((WARPS * ROWS * 130 + ROWS * 128) * 4 <= C::RING, "the join fits the ring");
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = l[nt][j];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int row = nt * 8 + 2 * ti + j;
      if (gi == 0) {
        part_m[warp * ROWS + row] = m[nt][j];
        part_l[warp * ROWS + row] = sum;
      }
      float4* dst = reinterpret_cast<float4*>(part_o + (warp * ROWS + row) * 128 + 16 * gi);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        dst[q] = make_float4(o[nt][2 * q][j], o[nt][2 * q][j + 2], o[nt][2 * q + 1][j], o[nt][2 * q + 1][j + 2]);
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < ROWS * 32; idx += WARPS * 32) {
    const int row = idx >> 5;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, part_m[w * ROWS + row]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = fast_exp2(part_m[w * ROWS + row] - mu);
      const float4 x = reinterpret_cast<const float4*>(part_o + (w * ROWS + row) * 128)[idx & 31];
      sum += f * part_l[w * ROWS + row];
      a.x += f * x.x;
      a.y += f * x.y;
      a.z += f * x.z;
      a.w += f * x.w;
    }
    reinterpret_cast<float4*>(cta_o + row * 128)[idx & 31] = a;
    if ((idx & 31) == 0) {
      join_m[row] = mx;
      join_l[row] = sum;
    }
  }
  if (ncta > 1)
    cluster_sync();
  else
    __syncthreads();
  for (int idx = rank * WARPS * 32 + threadIdx.x; idx < nrows * 32; idx += ncta * WARPS * 32) {
    const int row = idx >> 5;
    float mx = -INFINITY;
    for (int c = 0; c < ncta; ++c) mx = fmaxf(mx, ld_cluster_f(mapa_shared(join_m + row, c)));
    const float mu = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < ncta; ++c) {
      const float f = fast_exp2(ld_cluster_f(mapa_shared(join_m + row, c)) - mu);
      const float4 x = ld_cluster_f4(mapa_shared(cta_o + row * 128 + (idx & 31) * 4, c));
      sum += f * ld_cluster_f(mapa_shared(join_l + row, c));
      a.x += f * x.x;
      a.y += f * x.y;
      a.z += f * x.z;
      a.w += f * x.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no position is 0
    const int tok = row / nh, hd = row - tok * nh;
    uint16_t* dst = static_cast<uint16_t*>(p.out) + (start + t0 + tok) * p.ld_out + (kvh * g + h0 + hd) * 128 +
                    (idx & 31) * 4;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack16<F16>(a.x * inv, a.y * inv), pack16<F16>(a.z * inv, a.w * inv));
  }
  if (ncta > 1) cluster_sync();  // no CTA leaves while another reads its part
}

template <bool F16, int WARPS, int NT>
cudaError_t prepare_attend() {
  cudaError_t e = cudaFuncSetAttribute(k_cache_attend<F16, WARPS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       AttendCfg<WARPS, NT>::SMEM);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(k_cache_attend<F16, WARPS, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <bool F16, int WARPS, int NT>
cudaError_t launch_attend(const CacheAttnArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, long long items,
                          int ncta, int hpt, int head_tiles, int tpt, int* d_status, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ncta));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = AttendCfg<WARPS, NT>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ncta;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_cache_attend<F16, WARPS, NT>, tk, tv, a, hpt, head_tiles, tpt, d_status);
}

}  // namespace

int cache_write_launch(const CacheArgs& c, int f16, const int* offsets, long long rows, const void* k, long long ld_k,
                       const void* v, long long ld_v, int* d_status, cudaStream_t st) {
  const long long blocks = (rows / kPage + 2ll * c.nseq) * c.kv_heads;
  if (blocks > 0x7fffffffll) return -1;
  return static_cast<int>(launch_pdl(f16 ? k_cache_write<true> : k_cache_write<false>,
                                     dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, c, offsets, rows,
                                     static_cast<const uint16_t*>(k), ld_k, static_cast<const uint16_t*>(v), ld_v, d_status));
}

int cache_read_launch(const CacheArgs& c, int f16, const int* offsets, long long rows, void* k, long long ld_k,
                      void* v, long long ld_v, int* d_status, cudaStream_t st) {
  const long long blocks = (rows / kPage + 2ll * c.nseq) * c.kv_heads;
  if (blocks > 0x7fffffffll) return -1;
  return static_cast<int>(launch_pdl(f16 ? k_cache_read<true, false> : k_cache_read<false, false>,
                                     dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, c, offsets, rows,
                                     static_cast<uint16_t*>(k), ld_k, static_cast<uint16_t*>(v), ld_v, d_status));
}

static int dense_launch(const CacheArgs& c, int f16, void* k, void* v, int* d_status, cudaStream_t st) {
  const long long blocks = static_cast<long long>(c.nseq) * c.table_ld * c.kv_heads;
  if (blocks > 0x7fffffffll) return -1;
  const long long ld = static_cast<long long>(c.kv_heads) * 128;
  return static_cast<int>(launch_pdl(f16 ? k_cache_read<true, true> : k_cache_read<false, true>,
                                     dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, c, static_cast<const int*>(nullptr),
                                     0ll, static_cast<uint16_t*>(k), ld, static_cast<uint16_t*>(v), ld, d_status));
}

int cache_prepare() {
  cudaError_t e = prepare_attend<false, 4, 1>();
  if (e == cudaSuccess) e = prepare_attend<true, 4, 1>();
  if (e == cudaSuccess) e = prepare_attend<false, 4, 2>();
  if (e == cudaSuccess) e = prepare_attend<true, 4, 2>();
  return static_cast<int>(e);
}

// Rows (tokens times the query heads of a key/value head) a sequence, on average, beyond which the cache
// is turned into 16 bits once and read by the packed kernel's tensor-core tiles; up to it, the codes are
// read directly, 16 rows at a time.
constexpr long long kDenseRows = 64;

static bool dense_path(const CacheArgs& c, int heads, long long rows) {
  return rows * (heads / c.kv_heads) > kDenseRows * c.nseq;
}
static long long dense_rows(const CacheArgs& c) { return static_cast<long long>(c.nseq) * c.table_ld * kPage; }

size_t cache_attention_workspace(const CacheArgs& c, int heads, long long rows) {
  return dense_path(c, heads, rows) ? static_cast<size_t>(dense_rows(c)) * c.kv_heads * 128 * 2 * 2 : 0;
}

static int attend_launch(const CacheAttnArgs& a, int sms, int* d_status, cudaStream_t st) {
  const CacheArgs& c = a.c;
  const int g = a.heads / c.kv_heads;
  CUtensorMap tk, tv;
  const uint64_t d[3] = {128, kPage, static_cast<uint64_t>(c.pages) * c.kv_heads};
  const uint64_t s[2] = {128, PAGE_BYTES};
  const uint32_t b[3] = {128, kPage, 1};
  if (make_tmap(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.k, 3, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B) ||
      make_tmap(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.v, 3, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B))
    return -4;
  // 8 or 16 query rows a tile: 16 when the sequences' rows (on average) need more than 8
  const long long per = (a.rows + c.nseq - 1) / c.nseq;  // new tokens a sequence
  const int nt = per * g > 8 ? 2 : 1;
  const int hpt = g < 8 * nt ? g : 8 * nt, head_tiles = (g + hpt - 1) / hpt;
  const int room = 8 * nt / hpt;
  const int tpt = per < room ? static_cast<int>(per) : room;
  const long long items = (a.rows / tpt + (tpt == 1 ? 0 : c.nseq)) * head_tiles * c.kv_heads;
  // CTAs a cluster: as many as fill the SMs twice over, while each warp keeps a page to itself
  int ncta = 1;
  while (ncta < MAX_CLUSTER && items * ncta * 2 <= 2ll * sms && ncta * 4 < c.table_ld) ncta *= 2;
  if (items * ncta > 0x7fffffffll) return -1;
  cudaError_t e;
  if (a.f16)
    e = nt == 1 ? launch_attend<true, 4, 1>(a, tk, tv, items, ncta, hpt, head_tiles, tpt, d_status, st)
                : launch_attend<true, 4, 2>(a, tk, tv, items, ncta, hpt, head_tiles, tpt, d_status, st);
  else
    e = nt == 1 ? launch_attend<false, 4, 1>(a, tk, tv, items, ncta, hpt, head_tiles, tpt, d_status, st)
                : launch_attend<false, 4, 2>(a, tk, tv, items, ncta, hpt, head_tiles, tpt, d_status, st);
  return static_cast<int>(e);
}

int cache_attention(const CacheAttnArgs& a, void* ws, size_t ws_bytes, int sms, int* d_status, cudaStream_t st) {
  const CacheArgs& c = a.c;
  if (!dense_path(c, a.heads, a.rows)) return attend_launch(a, sms, d_status, st);
  if (ws_bytes < cache_attention_workspace(c, a.heads, a.rows) || dense_rows(c) > 0x7fffffffll) return -1;
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
  return packed_launch(p, d_status, st);
}

}  // namespace exn
