// rtg_qcache_*: the 8-bit key/value cache as a handle over device tensors
// (include/rtgpu.h); the kernels are in qcache.hip and qattn.hip.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <cmath>
#include <exception>
#include <memory>
#include <string>

#include "../../include/rtgpu.h"
#include "device_memory.h"
#include "qcache.h"

using namespace rtg;

struct rtg_qcache {
  QStore c;
  int device = 0;
  void* mem = nullptr;   // the store, lengths, error word and the attention's partial results
  int* len = nullptr;    // [n_seq]
  unsigned* tickets = nullptr;  // QTickets::count
  unsigned* err = nullptr;
  void* work = nullptr;
  ~rtg_qcache() {
    if (mem) (void)hipFree(mem);
  }
};

namespace {

rtg_result ok() { return rtg_result{true, nullptr}; }

rtg_result err(const char* f, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, f);
  vsnprintf(buf, sizeof buf, f, ap);
  va_end(ap);
  const size_t n = strlen(buf) + 1;
  char* s = static_cast<char*>(malloc(n));
  if (s) memcpy(s, buf, n);
  return rtg_result{false, s};
}

rtg_result hip_err(hipError_t e, const char* what) {
  (void)hipGetLastError();  // reported here, not by the caller's next check
  return err("HIP error in %s: %s", what, hipGetErrorString(e));
}

constexpr unsigned kNoErr = 0xFFFFFFFFu;
constexpr size_t kMaxGroup = 1024;
constexpr size_t kMaxRows = 4000000;  // of one sequence: a grid dimension of 65535 tiles of 64 tokens

// The handle's device as the current one for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (hipGetDevice(&before_) != hipSuccess) before_ = -1;
    if (before_ != device) status_ = hipSetDevice(device);
    set_ = before_ != device;
  }
  ~OnDevice() {
    if (set_ && before_ >= 0) (void)hipSetDevice(before_);
  }
  hipError_t status() const { return status_; }

 private:
  int before_ = -1;
  bool set_ = false;
  hipError_t status_ = hipSuccess;
};

// A kernel launch's own error (an earlier one of the caller's is not taken for it).
rtg_result launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ok() : hip_err(e, what);
}

bool type_of(rtg_dtype t, QType* q) {
  if (t == RTG_F32) *q = Q_F32;
  else if (t == RTG_BF16) *q = Q_BF16;
  else if (t == RTG_F16) *q = Q_F16;
  else return false;
  return true;
}

QRows rows(const rtg_rows* r) {
  QRows q;
  if (r) {
    q.p = r->data;
    q.seq = r->stride_seq;
    q.tok = r->stride_token;
    q.head = r->stride_head;
  }
  return q;
}

}  // namespace

extern "C" {

rtg_result rtg_qcache_new(size_t n_seq, size_t n_head, size_t head_dim, size_t capacity, size_t block,
                          rtg_qcache** out) {
  if (!out) return err("null argument");
  if (n_seq == 0 || n_head == 0 || capacity == 0) return err("n_seq, n_head and capacity must be >= 1");
  if (head_dim == 0 || head_dim > 128) return err("head_dim %zu is not supported (1 to 128)", head_dim);
  if (block != 16 && block != 32 && block != 64) return err("block %zu is not supported (16, 32 or 64)", block);
  if (capacity > kMaxRows) return err("capacity %zu exceeds %zu", capacity, kMaxRows);
  if (n_seq > 1000000 || n_head > 1000000 || n_seq * n_head > 1000000)
    return err("n_seq * n_head exceeds 1000000");
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n == 0)
    return err("no HIP device available: rtgpu requires an MI355X (gfx950) GPU");
  try {
    BesideCaptures beside;
    std::unique_ptr<rtg_qcache> q(new rtg_qcache());
    hipDeviceProp_t prop;
    if (hipGetDevice(&q->device) != hipSuccess || hipGetDeviceProperties(&prop, q->device) != hipSuccess)
      return err("hipGetDeviceProperties failed");
    if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
      return err("rtgpu is built for gfx950 (MI355X); found %s", prop.gcnArchName);
    qstore_shape(&q->c, (int)n_seq, (int)n_head, (int)head_dim, (int)capacity, (int)block);
    const size_t store = qstore_bytes(q->c), lens = (n_seq * 4 + 4 + 255) / 256 * 256;
    const size_t head = lens + (n_seq * (n_head + 1) * kQTicketStride * 4 + 255) / 256 * 256;
    hipError_t e = device_malloc(&q->mem, head + store + qattn_work_bytes(q->c.hdp));
    if (e != hipSuccess) return hip_err(e, "rtg_qcache_new");
    q->len = static_cast<int*>(q->mem);
    q->err = reinterpret_cast<unsigned*>(q->len + n_seq);
    q->tickets = reinterpret_cast<unsigned*>(static_cast<char*>(q->mem) + lens);
    qstore_place(&q->c, static_cast<char*>(q->mem) + head);
    q->work = static_cast<char*>(q->mem) + head + store;
    hipStream_t s = nullptr;  // (of its own: the default one may be what a capture waits for)
    e = hipStreamCreateWithFlags(&s, hipStreamNonBlocking);
    if (e == hipSuccess) e = hipMemsetAsync(q->mem, 0, head, s);
    if (e == hipSuccess) e = hipMemsetAsync(q->err, 0xFF, 4, s);
    if (e == hipSuccess) {
      qattn_work_clear(s, q->work, q->c.hdp);
      e = hipStreamSynchronize(s);
    }
    if (s) (void)hipStreamDestroy(s);
    if (e != hipSuccess) return hip_err(e, "rtg_qcache_new");
    *out = q.release();
  } catch (const std::exception& ex) {
    return err("internal error: %s", ex.what());
  }
  return ok();
}

void rtg_qcache_destroy(rtg_qcache* q) {
  if (!q) return;
  OnDevice dev(q->device);
  BesideCaptures beside;
  delete q;  // (hipFree waits for the device)
}

rtg_result rtg_qcache_append(rtg_qcache* q, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n_new,
                             const int32_t* counts, const int32_t* start, void* stream) {
  if (!q || !k || !v || (n_new && (!k->data || !v->data))) return err("null argument");
  QType t;
  if (!type_of(dtype, &t)) return err("rtg_qcache_append takes f32, bf16 or f16 rows");
  if (n_new > (size_t)q->c.capacity)
    return err("%zu new tokens exceed the cache's capacity %d", n_new, q->c.capacity);
  if (n_new == 0 && !start) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  (void)hipGetLastError();
  hipStream_t s = static_cast<hipStream_t>(stream);
  launch_q_append(s, q->c, QLen{q->len, 1}, QTickets{q->tickets, q->err}, t, rows(k), rows(v), (int)n_new, counts,
                  start);
  return launched("rtg_qcache_append");
}

rtg_result rtg_qcache_read(const rtg_qcache* q, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n,
                           const int32_t* first, void* stream) {
  if (!q) return err("null argument");
  QType t;
  if (!type_of(dtype, &t)) return err("rtg_qcache_read gives f32, bf16 or f16 rows");
  if (n > kMaxRows) return err("%zu rows exceed %zu", n, kMaxRows);
  const QRows kr = rows(k), vr = rows(v);
  if (n == 0 || (!kr.p && !vr.p)) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  (void)hipGetLastError();
  launch_q_read(static_cast<hipStream_t>(stream), q->c, QLen{q->len, 1}, t, kr, vr, (int)n, first);
  return launched("rtg_qcache_read");
}

rtg_result rtg_qcache_attend(rtg_qcache* q, rtg_dtype dtype, const rtg_rows* queries, size_t n_q, size_t n_q_head,
                             const int32_t* counts, float scale, const rtg_rows* out, void* stream) {
  if (!q || !queries || !out) return err("null argument");
  QType t;
  if (!type_of(dtype, &t)) return err("rtg_qcache_attend takes f32, bf16 or f16 rows");
  if (n_q_head == 0 || n_q_head % (size_t)q->c.n_head != 0)
    return err("%zu query heads are not a multiple of the cache's %d heads", n_q_head, q->c.n_head);
  if (n_q_head / q->c.n_head > kMaxGroup)
    return err("%zu query heads per key/value head exceed %zu", n_q_head / q->c.n_head, kMaxGroup);
  if (!std::isfinite(scale)) return err("scale must be finite");
  if (n_q > kMaxRows || n_q * (n_q_head / q->c.n_head) > kMaxRows)
    return err("%zu queries of %zu heads exceed %zu rows per key/value head", n_q, n_q_head, kMaxRows);
  if (n_q == 0) return ok();
  if (!queries->data || !out->data) return err("null argument");
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  (void)hipGetLastError();
  QOut o;
  o.rows = rows(out);
  launch_q_attend(static_cast<hipStream_t>(stream), q->c, QLen{q->len, 1}, 0, t, rows(queries), (int)n_q,
                  (int)n_q_head, counts, scale, o, q->work);
  return launched("rtg_qcache_attend");
}

rtg_result rtg_qcache_lengths(rtg_qcache* q, uint32_t* out, void* stream) {
  if (!q || !out) return err("null argument");
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (s && hipStreamIsCapturing(s, &capture) == hipSuccess && capture != hipStreamCaptureStatusNone)
    return err("rtg_qcache_lengths: the stream is being captured");  // (a copy would end the capture)
  unsigned bad = kNoErr;
  hipError_t e = hipMemcpyAsync(out, q->len, (size_t)q->c.n_seq * 4, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipMemcpyAsync(&bad, q->err, 4, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e == hipSuccess && bad != kNoErr) {
    e = hipMemsetAsync(q->err, 0xFF, 4, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
  }
  if (e != hipSuccess) return hip_err(e, "rtg_qcache_lengths");
  if (bad == kNoErr) return ok();
  if (bad % 4 == 1) return err("sequence %u: an append's start is not within the sequence", bad / 4);
  return err("sequence %u: an append exceeds the cache's capacity %d", bad / 4, q->c.capacity);
}

}  // extern "C"
