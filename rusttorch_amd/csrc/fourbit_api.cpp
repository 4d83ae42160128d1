// rtg_fourbit_*: the 4-bit key/value cache as a handle over device tensors, and
// rtg_attend_packed: attention over packed prompts (include/rtgpu.h); the kernels
// are in fourbit.hip, fourbit_attn.hip and attn_tile.hip.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <cmath>
#include <exception>
#include <memory>

#include "../../include/rtgpu.h"
#include "device_memory.h"
#include "fourbit.h"

using namespace rtg;

struct rtg_fourbit {
  FStore c;
  int device = 0;
  void* mem = nullptr;          // lengths, error word, tickets, the store, attention's partial results
  int* len = nullptr;           // [n_seq]
  QTickets tickets;
  void* work = nullptr;
  ~rtg_fourbit() {
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
constexpr size_t kMaxRows = 4000000;  // of one sequence

// The handle's device as the current one for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (hipGetDevice(&before_) != hipSuccess) before_ = -1;
    if (before_ != device) status_ = hipSetDevice(device);
    set_ = before_ != device;
    (void)hipGetLastError();  // (an earlier error of the caller's is not taken for a launch's)
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

rtg_result this_gpu(int* device) {
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n == 0)
    return err("no HIP device available: rtgpu requires an MI355X (gfx950) GPU");
  hipDeviceProp_t prop;
  if (hipGetDevice(device) != hipSuccess || hipGetDeviceProperties(&prop, *device) != hipSuccess)
    return err("hipGetDeviceProperties failed");
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    return err("rtgpu is built for gfx950 (MI355X); found %s", prop.gcnArchName);
  return ok();
}

}  // namespace

extern "C" {

rtg_result rtg_fourbit_new(size_t n_seq, size_t n_head, size_t head_dim, size_t capacity, rtg_fourbit** out) {
  if (!out) return err("null argument");
  if (n_seq == 0 || n_head == 0 || capacity == 0) return err("n_seq, n_head and capacity must be >= 1");
  if (head_dim == 0 || head_dim > 128) return err("head_dim %zu is not supported (1 to 128)", head_dim);
  if (capacity > kMaxRows) return err("capacity %zu exceeds %zu", capacity, kMaxRows);
  if (n_seq > 1000000 || n_head > 1000000 || n_seq * n_head > 1000000)
    return err("n_seq * n_head exceeds 1000000");
  int device = 0;
  const rtg_result gpu = this_gpu(&device);
  if (!gpu.success) return gpu;
  try {
    BesideCaptures beside;
    std::unique_ptr<rtg_fourbit> q(new rtg_fourbit());
    q->device = device;
    fstore_shape(&q->c, (int)n_seq, (int)n_head, (int)head_dim, (int)capacity);
    const size_t lens = (n_seq * 4 + 4 + 255) / 256 * 256, head = lens + n_seq * kQTicketStride * 4;
    hipError_t e = device_malloc(&q->mem, (head + 255) / 256 * 256 + q->c.sizes().bytes() + fattn_work_bytes(q->c));
    if (e != hipSuccess) return hip_err(e, "rtg_fourbit_new");
    char* mem = static_cast<char*>(q->mem);
    q->len = static_cast<int*>(q->mem);
    q->tickets.err = reinterpret_cast<unsigned*>(q->len + n_seq);
    q->tickets.count = reinterpret_cast<unsigned*>(mem + lens);
    mem += (head + 255) / 256 * 256;
    fstore_place(&q->c, mem);
    q->work = mem + q->c.sizes().bytes();
    hipStream_t s = nullptr;  // (of its own: the default one may be what a capture waits for)
    e = hipStreamCreateWithFlags(&s, hipStreamNonBlocking);
    if (e == hipSuccess) e = hipMemsetAsync(q->mem, 0, head, s);
    if (e == hipSuccess) e = hipMemsetAsync(q->tickets.err, 0xFF, 4, s);
    if (e == hipSuccess) {
      fattn_work_clear(s, q->work);
      e = hipStreamSynchronize(s);
    }
    if (s) (void)hipStreamDestroy(s);
    if (e != hipSuccess) return hip_err(e, "rtg_fourbit_new");
    *out = q.release();
  } catch (const std::exception& ex) {
    return err("internal error: %s", ex.what());
  }
  return ok();
}

void rtg_fourbit_destroy(rtg_fourbit* q) {
  if (!q) return;
  OnDevice dev(q->device);
  BesideCaptures beside;
  delete q;  // (hipFree waits for the device)
}

rtg_result rtg_fourbit_append(rtg_fourbit* q, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n_new,
                              const int32_t* counts, const int32_t* start, void* stream) {
  if (!q || !k || !v || (n_new && (!k->data || !v->data))) return err("null argument");
  QType t;
  if (!type_of(dtype, &t)) return err("rtg_fourbit_append takes f32, bf16 or f16 rows");
  if (n_new > (size_t)q->c.capacity)
    return err("%zu new tokens exceed the cache's capacity %d", n_new, q->c.capacity);
  if (n_new == 0 && !start) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  launch_f_append(static_cast<hipStream_t>(stream), q->c, q->len, q->tickets, t, rows(k), rows(v), (int)n_new, counts,
                  start);
  return launched("rtg_fourbit_append");
}

rtg_result rtg_fourbit_read(const rtg_fourbit* q, rtg_dtype dtype, const rtg_rows* k, const rtg_rows* v, size_t n,
                            const int32_t* first, void* stream) {
  if (!q) return err("null argument");
  QType t;
  if (!type_of(dtype, &t)) return err("rtg_fourbit_read gives f32, bf16 or f16 rows");
  if (n > kMaxRows) return err("%zu rows exceed %zu", n, kMaxRows);
  const QRows kr = rows(k), vr = rows(v);
  if (n == 0 || (!kr.p && !vr.p)) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  launch_f_read(static_cast<hipStream_t>(stream), q->c, q->len, t, kr, vr, (int)n, first);
  return launched("rtg_fourbit_read");
}

rtg_result rtg_fourbit_attend(rtg_fourbit* q, rtg_dtype dtype, const rtg_rows* queries, size_t n_q, size_t n_q_head,
                              const int32_t* counts, float scale, const rtg_rows* out, float* stats, float decay,
                              void* stream) {
  if (!q || !queries || !out) return err("null argument");
  FAttn f;
  if (!type_of(dtype, &f.type)) return err("rtg_fourbit_attend takes f32, bf16 or f16 rows");
  if (n_q_head == 0 || n_q_head % (size_t)q->c.n_head != 0)
    return err("%zu query heads are not a multiple of the cache's %d heads", n_q_head, q->c.n_head);
  if (n_q_head / q->c.n_head > kMaxGroup)
    return err("%zu query heads per key/value head exceed %zu", n_q_head / q->c.n_head, kMaxGroup);
  if (!std::isfinite(scale)) return err("scale must be finite");
  if (stats && !(decay >= 0.f && decay <= 1.f)) return err("decay must be within 0 .. 1");
  if (n_q > kMaxRows || n_q * (n_q_head / q->c.n_head) > kMaxRows)
    return err("%zu queries of %zu heads exceed %zu rows per key/value head", n_q, n_q_head, kMaxRows);
  if (n_q == 0 && !stats) return ok();
  if (n_q && (!queries->data || !out->data)) return err("null argument");
  f.c = q->c;
  f.len = q->len;
  f.q = rows(queries);
  f.out = rows(out);
  f.n_q = (int)n_q;
  f.n_q_head = (int)n_q_head;
  f.counts = counts;
  f.scale = scale;
  f.stats = stats;
  f.work = q->work;
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_q) launch_f_attend(s, f);
  if (stats) launch_f_weigh(s, f, decay);
  return launched("rtg_fourbit_attend");
}

rtg_result rtg_fourbit_weights(const rtg_fourbit* q, float* out, size_t n, void* stream) {
  if (!q || (n && !out)) return err("null argument");
  if (n > kMaxRows) return err("%zu rows exceed %zu", n, kMaxRows);
  if (n == 0) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  launch_f_weights(static_cast<hipStream_t>(stream), q->c, q->len, out, (int)n);
  return launched("rtg_fourbit_weights");
}

rtg_result rtg_fourbit_add_weights(rtg_fourbit* q, const float* x, size_t n, void* stream) {
  if (!q || (n && !x)) return err("null argument");
  if (n > kMaxRows) return err("%zu rows exceed %zu", n, kMaxRows);
  if (n == 0) return ok();
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  launch_f_add_weights(static_cast<hipStream_t>(stream), q->c, q->len, x, (int)n);
  return launched("rtg_fourbit_add_weights");
}

rtg_result rtg_fourbit_evict(rtg_fourbit* q, size_t keep, size_t recent, int32_t* kept, void* stream) {
  if (!q || !kept) return err("null argument");
  if (keep == 0) return err("keep must be >= 1");
  if (keep > (size_t)q->c.capacity) return err("keep %zu exceeds the cache's capacity %d", keep, q->c.capacity);
  if (recent > keep) return err("recent %zu exceeds keep %zu", recent, keep);
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  launch_f_evict(static_cast<hipStream_t>(stream), q->c, q->len, q->tickets, (int)keep, (int)recent, kept);
  return launched("rtg_fourbit_evict");
}

rtg_result rtg_fourbit_lengths(rtg_fourbit* q, uint32_t* out, void* stream) {
  if (!q || !out) return err("null argument");
  OnDevice dev(q->device);
  if (dev.status() != hipSuccess) return hip_err(dev.status(), "hipSetDevice");
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (s && hipStreamIsCapturing(s, &capture) == hipSuccess && capture != hipStreamCaptureStatusNone)
    return err("rtg_fourbit_lengths: the stream is being captured");  // (a copy would end the capture)
  unsigned bad = kNoErr;
  hipError_t e = hipMemcpyAsync(out, q->len, (size_t)q->c.n_seq * 4, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipMemcpyAsync(&bad, q->tickets.err, 4, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e == hipSuccess && bad != kNoErr) {
    e = hipMemsetAsync(q->tickets.err, 0xFF, 4, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
  }
  if (e != hipSuccess) return hip_err(e, "rtg_fourbit_lengths");
  if (bad == kNoErr) return ok();
  if (bad % 4 == 1) return err("sequence %u: an append's start is not within the sequence", bad / 4);
  return err("sequence %u: an append exceeds the cache's capacity %d", bad / 4, q->c.capacity);
}

rtg_result rtg_attend_packed(rtg_dtype dtype, const rtg_rows* q, const rtg_rows* k, const rtg_rows* v, size_t n_rows,
                             size_t n_q_head, size_t n_head, size_t head_dim, const int32_t* offsets, size_t n_seq,
                             float scale, const rtg_rows* out, void* stream) {
  if (!q || !k || !v || !out || !offsets) return err("null argument");
  PAttn p;
  if (!type_of(dtype, &p.type)) return err("rtg_attend_packed takes f32, bf16 or f16 rows");
  if (head_dim == 0 || head_dim > 128) return err("head_dim %zu is not supported (1 to 128)", head_dim);
  if (n_head == 0 || n_q_head == 0 || n_q_head % n_head != 0)
    return err("%zu query heads are not a multiple of %zu heads", n_q_head, n_head);
  if (n_q_head / n_head > kMaxGroup)
    return err("%zu query heads per key/value head exceed %zu", n_q_head / n_head, kMaxGroup);
  if (n_seq == 0 || n_seq > 1000000) return err("n_seq must be within 1 .. 1000000");
  // (32-bit numbers of rows and heads; a grid of 2^32 threads)
  constexpr size_t kMostRows = 100000000, kMostPairs = 1600000000, kMostGroups = 8000000;
  if (n_rows > kMostRows || n_q_head > 1000000 || n_rows * n_q_head > kMostPairs)
    return err("%zu rows of %zu heads exceed %zu", n_rows, n_q_head, kMostPairs);
  if ((n_rows * (n_q_head / n_head) / 128 + 1 + n_seq) * n_head > kMostGroups)
    return err("%zu rows and %zu sequences of %zu heads are too many", n_rows, n_seq, n_head);
  if (!std::isfinite(scale)) return err("scale must be finite");
  if (n_rows == 0) return ok();
  if (!q->data || !k->data || !v->data || !out->data) return err("null argument");
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess)
    return err("no HIP device available: rtgpu requires an MI355X (gfx950) GPU");
  (void)hipGetLastError();
  p.q = rows(q);
  p.k = rows(k);
  p.v = rows(v);
  p.out = rows(out);
  p.q.seq = p.k.seq = p.v.seq = p.out.seq = 0;
  p.n_rows = (int)n_rows;
  p.n_seq = (int)n_seq;
  p.n_head = (int)n_head;
  p.n_q_head = (int)n_q_head;
  p.hd = (int)head_dim;
  p.offsets = offsets;
  p.scale = scale;
  launch_packed_attend(static_cast<hipStream_t>(stream), p);
  return launched("rtg_attend_packed");
}

}  // extern "C"
