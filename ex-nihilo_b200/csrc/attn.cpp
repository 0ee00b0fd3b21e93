// attn.cpp -- the host side of exn_attn_* (include/exn_b200.h): the checks of
// the attention operators' arguments and their launches on the caller's stream.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <new>

#include "../../include/exn_b200.h"
#include "../../include/exn_b200_testing.h"
#include "exn_internal.h"

using namespace exn;

struct exn_attn {
  int device = 0, sms = 0, fit[3] = {0, 0, 0};
  int* d_status = nullptr;  // what the kernels set, and behind it what exn_attn_sync took of it
  char err[512] = "";  // no allocation, so no exception either, on the way to the caller
};

namespace {

thread_local char g_attn_open_error[512];

int afail(exn_attn* a, int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(a ? a->err : g_attn_open_error, 512, fmt, ap);
  va_end(ap);
  return code;
}

#define ACK(call)                                                                                       \
  do {                                                                                                  \
    cudaError_t e_ = (call);                                                                            \
    if (e_ != cudaSuccess)                                                                              \
      return afail(a, e_ == cudaErrorMemoryAllocation ? EXN_ENOMEM : EXN_ECUDA, "%s: %s (%s:%d)", #call, \
                   cudaGetErrorString(e_), __FILE__, __LINE__);                                         \
  } while (0)

// the handle's device current for the call, the caller's again after it
struct OnDevice {
  int before = -1;
  cudaError_t rc;
  explicit OnDevice(int device) {
    rc = cudaGetDevice(&before);
    if (rc == cudaSuccess && before != device) rc = cudaSetDevice(device);
    else if (rc == cudaSuccess) before = -1;  // nothing to put back
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

constexpr int64_t kMaxRows = 0x7fffffff;

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_type(exn_attn* a, const char* fn, int type) {
  if (type != EXN_GGML_BF16 && type != EXN_GGML_F16)
    return afail(a, EXN_EINVAL, "%s: type %d is neither EXN_GGML_BF16 nor EXN_GGML_F16", fn, type);
  return EXN_OK;
}

int check_heads(exn_attn* a, const char* fn, int heads, int kv_heads) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > 128 || heads > 65536)
    return afail(a, EXN_EINVAL, "%s: %d query heads on %d key/value heads (a multiple, at most 128 times)", fn, heads, kv_heads);
  return EXN_OK;
}

// a packed matrix of HEADS heads: its row stride (0: contiguous) and base; *LD is filled in
int check_matrix(exn_attn* a, const char* fn, const char* what, const void* p, int64_t* ld, int heads) {
  const int64_t w = static_cast<int64_t>(heads) * 128;
  if (*ld == 0) *ld = w;
  if (!p) return afail(a, EXN_EINVAL, "%s: %s is null", fn, what);
  if (!aligned(p, 16)) return afail(a, EXN_EINVAL, "%s: %s is not 16-byte aligned", fn, what);
  if (*ld < w || *ld % 8 || *ld > (1ll << 36))
    return afail(a, EXN_EINVAL, "%s: the row stride of %s is %lld elements (at least %lld, a multiple of 8)", fn, what,
                 static_cast<long long>(*ld), static_cast<long long>(w));
  return EXN_OK;
}

int check_rows(exn_attn* a, const char* fn, int nseq, int64_t rows, const void* offsets) {
  if (nseq < 0 || rows < 0 || rows > kMaxRows)
    return afail(a, EXN_EINVAL, "%s: %d sequences, %lld rows", fn, nseq, static_cast<long long>(rows));
  if (nseq > 0 && !offsets) return afail(a, EXN_EINVAL, "%s: the offsets are null", fn);
  if (!aligned(offsets, 4)) return afail(a, EXN_EINVAL, "%s: the offsets are not 4-byte aligned", fn);
  return EXN_OK;
}

int check_scale(exn_attn* a, const char* fn, double scale, float* log2) {
  const double s = scale == 0 ? 1.0 / std::sqrt(128.0) : scale;
  *log2 = static_cast<float>(s * 1.4426950408889634);
  if (!(s > 0) || !std::isfinite(*log2) || *log2 <= 0.f)
    return afail(a, EXN_EINVAL, "%s: scale %g (0, or positive and finite)", fn, scale);
  return EXN_OK;
}

int check_cache(exn_attn* a, const char* fn, const exn_kv_cache* c, CacheArgs* out) {
  if (!c) return afail(a, EXN_EINVAL, "%s: the cache is null", fn);
  if (c->kv_heads <= 0 || c->kv_heads > 65536 || c->nseq < 0 || c->pages <= 0 || c->table_ld <= 0 ||
      c->table_ld > kMaxRows / kPage || static_cast<int64_t>(c->pages) * c->kv_heads > kMaxRows)
    return afail(a, EXN_EINVAL, "%s: a cache of %d heads, %d sequences, %d pages, %d table entries a sequence", fn,
                 c->kv_heads, c->nseq, c->pages, c->table_ld);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || (c->nseq > 0 && (!c->table || !c->lens)))
    return afail(a, EXN_EINVAL, "%s: the cache has a null pointer", fn);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->table, 4) || !aligned(c->lens, 4))
    return afail(a, EXN_EINVAL, "%s: the cache's codes are not 16-byte or its tables not 4-byte aligned", fn);
  out->kv_heads = c->kv_heads;
  out->nseq = c->nseq;
  out->pages = c->pages;
  out->table_ld = c->table_ld;
  out->k = c->k;
  out->v = c->v;
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->table = c->table;
  out->lens = c->lens;
  return EXN_OK;
}

int launched(exn_attn* a, const char* fn, int r) {
  if (r == 0) return EXN_OK;
  if (r == -1) return afail(a, EXN_EINVAL, "%s: too many tiles for one launch", fn);
  if (r == -4) return afail(a, EXN_EINVAL, "%s: the tensors cannot be described to the TMA unit (size or stride)", fn);
  return afail(a, EXN_ECUDA, "%s: launch failed: %s", fn, cudaGetErrorString(static_cast<cudaError_t>(r)));
}

// what the kernels' status word says; a kernel that gave up comes first, since then nothing is to be trusted
int report(exn_attn* a, int s) {
  if (!s) return EXN_OK;
  if (s & ~STATUS_BAD_ARG_BIT)
    return afail(a, EXN_ETIMEOUT, "a kernel gave up waiting on its pipeline (status 0x%x)%s", s,
                 s & STATUS_BAD_ARG_BIT ? ", and one met offsets, lengths or pages out of range" : "");
  return afail(a, EXN_EINVAL,
               "a kernel met offsets that decrease or pass the rows, lengths shorter than a sequence's rows, or "
               "table entries that are not pages of the pool; it left them out");
}

}  // namespace

extern "C" {

int exn_attn_open(int device, exn_attn** out) {
  if (!out) return afail(nullptr, EXN_EINVAL, "exn_attn_open: null argument");
  *out = nullptr;
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev)
    return afail(nullptr, EXN_ECUDA, "exn_attn_open: no CUDA device %d", device);
  cudaDeviceProp prop;
  if (cudaGetDeviceProperties(&prop, device) != cudaSuccess)
    return afail(nullptr, EXN_ECUDA, "exn_attn_open: cannot query device %d", device);
  if (prop.major != 10)
    return afail(nullptr, EXN_EUNSUPPORTED, "exn_attn_open: device %d is sm_%d%d; this library is built for sm_100a",
                 device, prop.major, prop.minor);
  exn_attn* a = new (std::nothrow) exn_attn();
  if (!a) return afail(nullptr, EXN_ENOMEM, "exn_attn_open: out of memory");
  a->device = device;
  a->sms = prop.multiProcessorCount;
  const int rc = [&]() -> int {
    OnDevice on(device);
    ACK(on.rc);
    ACK(cudaMalloc(&a->d_status, 2 * sizeof(int)));
    ACK(cudaMemset(a->d_status, 0, 2 * sizeof(int)));
    ACK(static_cast<cudaError_t>(packed_prepare(a->fit)));
    ACK(static_cast<cudaError_t>(cache_prepare()));
    return EXN_OK;
  }();
  if (rc) {
    memcpy(g_attn_open_error, a->err, sizeof a->err);
    exn_attn_close(a);
    return rc;
  }
  *out = a;
  return EXN_OK;
}

void exn_attn_close(exn_attn* a) {
  if (!a) return;
  {
    OnDevice on(a->device);
    if (a->d_status) cudaFree(a->d_status);  // waits for the device's queued kernels
  }
  delete a;
}

const char* exn_attn_last_error(const exn_attn* a) { return a ? a->err : g_attn_open_error; }

int exn_attn_sync(exn_attn* a, void* stream) {
  if (!a) return afail(a, EXN_EINVAL, "exn_attn_sync: null handle");
  OnDevice on(a->device);
  ACK(on.rc);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int s = 0;
  ACK(static_cast<cudaError_t>(status_take_launch(a->d_status, st)));
  ACK(cudaMemcpyAsync(&s, a->d_status + 1, sizeof s, cudaMemcpyDeviceToHost, st));
  ACK(cudaStreamSynchronize(st));
  return report(a, s);
}

int exn_attn_packed(exn_attn* a, int type, int heads, int kv_heads, int nseq, const int32_t* q_offsets,
                    const int32_t* kv_offsets, int64_t rows, int64_t kv_rows, const void* q, int64_t ld_q,
                    const void* k, int64_t ld_k, const void* v, int64_t ld_v, void* out, int64_t ld_out,
                    double scale, void* stream) {
  static const char fn[] = "exn_attn_packed";
  if (!a) return afail(a, EXN_EINVAL, "%s: null handle", fn);
  int rc;
  PackedArgs p;
  if ((rc = check_type(a, fn, type)) || (rc = check_heads(a, fn, heads, kv_heads)) ||
      (rc = check_rows(a, fn, nseq, rows, q_offsets)) || (rc = check_scale(a, fn, scale, &p.scale_log2)))
    return rc;
  if (!kv_offsets && kv_rows != rows)
    return afail(a, EXN_EINVAL, "%s: %lld query rows, %lld key rows, and one set of offsets", fn,
                 static_cast<long long>(rows), static_cast<long long>(kv_rows));
  if (kv_rows < 0 || kv_rows > kMaxRows || !aligned(kv_offsets, 4))
    return afail(a, EXN_EINVAL, "%s: %lld key rows, or their offsets are not 4-byte aligned", fn, static_cast<long long>(kv_rows));
  if (nseq == 0 || rows == 0) return EXN_OK;
  if ((rc = check_matrix(a, fn, "q", q, &ld_q, heads)) || (rc = check_matrix(a, fn, "out", out, &ld_out, heads)))
    return rc;
  if (kv_rows > 0 && ((rc = check_matrix(a, fn, "k", k, &ld_k, kv_heads)) || (rc = check_matrix(a, fn, "v", v, &ld_v, kv_heads))))
    return rc;
  if (kv_rows == 0) {  // no key anywhere: q stands in for the tensors, which are not read
    k = v = q;
    ld_k = ld_v = ld_q;
  }
  OnDevice on(a->device);
  ACK(on.rc);
  p.f16 = type == EXN_GGML_F16;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.nseq = nseq;
  p.q_offsets = q_offsets;
  p.kv_offsets = kv_offsets ? kv_offsets : q_offsets;
  p.rows = rows;
  p.kv_rows = kv_rows;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.ld_q = ld_q;
  p.ld_k = ld_k;
  p.ld_v = ld_v;
  p.ld_out = ld_out;
  for (int i = 0; i < 3; ++i) p.fit[i] = a->fit[i];
  return launched(a, fn, packed_launch(p, a->d_status, static_cast<cudaStream_t>(stream)));
}

int exn_attn_cache_write(exn_attn* a, const exn_kv_cache* cache, int type, const int32_t* offsets, int64_t rows,
                         const void* k, int64_t ld_k, const void* v, int64_t ld_v, void* stream) {
  static const char fn[] = "exn_attn_cache_write";
  if (!a) return afail(a, EXN_EINVAL, "%s: null handle", fn);
  int rc;
  CacheArgs c;
  if ((rc = check_type(a, fn, type)) || (rc = check_cache(a, fn, cache, &c)) ||
      (rc = check_rows(a, fn, c.nseq, rows, offsets)))
    return rc;
  if (c.nseq == 0 || rows == 0) return EXN_OK;
  if ((rc = check_matrix(a, fn, "k", k, &ld_k, c.kv_heads)) || (rc = check_matrix(a, fn, "v", v, &ld_v, c.kv_heads)))
    return rc;
  OnDevice on(a->device);
  ACK(on.rc);
  return launched(a, fn, cache_write_launch(c, type == EXN_GGML_F16, offsets, rows, k, ld_k, v, ld_v, a->d_status,
                                            static_cast<cudaStream_t>(stream)));
}

int exn_attn_cache_read(exn_attn* a, const exn_kv_cache* cache, int type, const int32_t* offsets, int64_t rows,
                        void* k, int64_t ld_k, void* v, int64_t ld_v, void* stream) {
  static const char fn[] = "exn_attn_cache_read";
  if (!a) return afail(a, EXN_EINVAL, "%s: null handle", fn);
  int rc;
  CacheArgs c;
  if ((rc = check_type(a, fn, type)) || (rc = check_cache(a, fn, cache, &c)) ||
      (rc = check_rows(a, fn, c.nseq, rows, offsets)))
    return rc;
  if (c.nseq == 0 || rows == 0) return EXN_OK;
  if ((rc = check_matrix(a, fn, "k", k, &ld_k, c.kv_heads)) || (rc = check_matrix(a, fn, "v", v, &ld_v, c.kv_heads)))
    return rc;
  OnDevice on(a->device);
  ACK(on.rc);
  return launched(a, fn, cache_read_launch(c, type == EXN_GGML_F16, offsets, rows, k, ld_k, v, ld_v, a->d_status,
                                           static_cast<cudaStream_t>(stream)));
}

int exn_attn_cache_workspace(exn_attn* a, const exn_kv_cache* cache, int heads, int64_t rows, size_t* bytes) {
  static const char fn[] = "exn_attn_cache_workspace";
  if (!a) return afail(a, EXN_EINVAL, "%s: null handle", fn);
  int rc;
  CacheArgs c;
  if ((rc = check_cache(a, fn, cache, &c)) || (rc = check_heads(a, fn, heads, c.kv_heads))) return rc;
  if (!bytes || rows < 0 || rows > kMaxRows) return afail(a, EXN_EINVAL, "%s: null result, or %lld rows", fn, static_cast<long long>(rows));
  *bytes = c.nseq ? cache_attention_workspace(c, heads, rows, a->sms) : 0;
  return EXN_OK;
}

int exn_attn_cache_attend(exn_attn* a, const exn_kv_cache* cache, int type, int heads, const int32_t* offsets,
                          int64_t rows, const void* q, int64_t ld_q, void* out, int64_t ld_out, double scale,
                          void* workspace, size_t workspace_bytes, void* stream) {
  static const char fn[] = "exn_attn_cache_attend";
  if (!a) return afail(a, EXN_EINVAL, "%s: null handle", fn);
  int rc;
  CacheAttnArgs p;
  if ((rc = check_type(a, fn, type)) || (rc = check_cache(a, fn, cache, &p.c)) ||
      (rc = check_heads(a, fn, heads, p.c.kv_heads)) || (rc = check_rows(a, fn, p.c.nseq, rows, offsets)) ||
      (rc = check_scale(a, fn, scale, &p.scale_log2)))
    return rc;
  if (p.c.nseq == 0 || rows == 0) return EXN_OK;
  if ((rc = check_matrix(a, fn, "q", q, &ld_q, heads)) || (rc = check_matrix(a, fn, "out", out, &ld_out, heads)))
    return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = cache_attention_workspace(p.c, heads, rows, a->sms);
  if (need > workspace_bytes || (need && !workspace))
    return afail(a, EXN_EINVAL, "%s: a workspace of %zu bytes, %zu needed", fn, workspace ? workspace_bytes : 0, need);
  if (need && !aligned(workspace, 256)) return afail(a, EXN_EINVAL, "%s: the workspace is not 256-byte aligned", fn);
  OnDevice on(a->device);
  ACK(on.rc);
  p.f16 = type == EXN_GGML_F16;
  p.heads = heads;
  p.offsets = offsets;
  p.rows = rows;
  p.q = q;
  p.ld_q = ld_q;
  p.out = out;
  p.ld_out = ld_out;
  return launched(a, fn, cache_attention(p, workspace, workspace_bytes, a->sms, a->fit, a->d_status, st));
}

// include/exn_b200_testing.h
int exn_test_attn_report(int status, char* text, int n) {
  exn_attn a;
  const int rc = report(&a, status);
  snprintf(text, n, "%s", a.err);
  return rc;
}

}  // extern "C"
