// C ABI of the losses on policy logits and of the gradient clipping
// (include/mfhip.h): argument checks, the device and stream of a call, and
// the launches.  Shapes are checked before any device is touched.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/mfhip.h"
#include "learn_ranges.h"
#include "mfh_kernels.h"
#include "mfh_status.h"

struct mfh_grad_set {
  int device = 0;
  std::int64_t n_chunks = 0;
  bool past = false;                 // too large for the caches
  mfh::GradChunk *chunks = nullptr;  // device memory, read only
  std::vector<mfh::ByteRange> memory;  // of every src and dst
};

namespace {

using mfh::SetError;

int HipError(const char *fn, const char *what, hipError_t e) {
  (void)hipGetLastError();
  return SetError(MFH_ERR_HIP, std::string(fn) + ": " + what + ": " + hipGetErrorString(e));
}

int Invalid(const char *fn, const char *what) {
  return SetError(MFH_ERR_INVALID, std::string(fn) + ": " + what);
}

bool Aligned(const void *p, std::uintptr_t bytes) {
  return reinterpret_cast<std::uintptr_t>(p) % bytes == 0;
}

// Makes `device` current for a call and puts the caller's device back.
class OnDevice {
 public:
  ~OnDevice() {
    if (before_ >= 0)
      (void)hipSetDevice(before_);
  }
  hipError_t Set(int device) {
    int now = 0;
    hipError_t e = hipGetDevice(&now);
    if (e != hipSuccess || now == device)
      return e;
    e = hipSetDevice(device);
    if (e == hipSuccess)
      before_ = now;
    return e;
  }

 private:
  int before_ = -1;
};

// Whether device `dev` is a gfx950, looked up once per device.
bool IsGfx950(int dev) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices] = {};  // 0 unknown, 1 yes, 2 no
  if (dev < 0 || dev >= kMaxDevices)
    return false;
  int k = known[dev].load(std::memory_order_relaxed);
  if (k == 0) {
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, dev) != hipSuccess) {
      (void)hipGetLastError();
      return false;
    }
    k = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
    known[dev].store(k, std::memory_order_relaxed);
  }
  return k == 1;
}

int NeedDevice(const char *fn, int dev) {
  static std::atomic<int> count{-1};
  int n = count.load(std::memory_order_relaxed);
  if (n < 0) {
    if (hipGetDeviceCount(&n) != hipSuccess) {
      (void)hipGetLastError();
      n = 0;
    }
    count.store(n, std::memory_order_relaxed);
  }
  if (n <= 0)
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": no HIP device available");
  if (dev >= n)
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": device ordinal out of range");
  return MFH_OK;
}

// The device of `p`; an error if it is not device memory, or (want >= 0)
// another device's.
int PointerDevice(const char *fn, const char *name, const void *p, int want, int *dev) {
  hipPointerAttribute_t attr;
  const hipError_t e = hipPointerGetAttributes(&attr, p);
  if (e != hipSuccess)
    (void)hipGetLastError();
  if (e != hipSuccess || (attr.type != hipMemoryTypeDevice && attr.type != hipMemoryTypeManaged))
    return Invalid(fn, (std::string(name) + " is not device memory").c_str());
  if (want >= 0 && attr.device != want)
    return Invalid(fn, (std::string(name) + " is on another device").c_str());
  if (dev)
    *dev = attr.device;
  return MFH_OK;
}

int StreamDevice(const char *fn, hipStream_t stream, int device) {
  // The standing streams belong to the device that is current at the launch.
  if (!stream || stream == hipStreamPerThread || stream == hipStreamLegacy)
    return MFH_OK;
  hipDevice_t dev = 0;
  const hipError_t e = hipStreamGetDevice(stream, &dev);
  if (e != hipSuccess)
    return HipError(fn, "stream", e);
  if (dev != device)
    return Invalid(fn, "the stream is another device's");
  return MFH_OK;
}

struct Named {
  const char *name;
  const void *p;
};

// Device, stream and pointers of a call: sets `on` to the device of the
// first pointer (or `want`), and checks the rest against it.
template <size_t N>
int Enter(const char *fn, int want, const Named (&ptrs)[N], hipStream_t stream, OnDevice *on) {
  int rc = NeedDevice(fn, want);
  if (rc != MFH_OK)
    return rc;
  int dev = want >= 0 ? want : -1;
  for (const Named &n : ptrs) {
    if (!n.p)
      continue;
    int d = dev;
    rc = PointerDevice(fn, n.name, n.p, dev, &d);
    if (rc != MFH_OK)
      return rc;
    dev = d;
  }
  if (!IsGfx950(dev))
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": the device is not gfx950 (MI355X)");
  rc = StreamDevice(fn, stream, dev);
  if (rc != MFH_OK)
    return rc;
  const hipError_t e = on->Set(dev);
  return e == hipSuccess ? MFH_OK : HipError(fn, "hipSetDevice", e);
}

// An array without gaps.
mfh::Span Flat(const char *name, const void *p, std::int64_t bytes, bool written) {
  return {name, p, 1, bytes, bytes, written, false};
}

// Rows of the logits' shape.
mfh::Span Rows(const char *name, const void *p, const mfh_policy_rows *r, std::int64_t stride,
               bool written) {
  const std::int64_t es = mfh::DTypeBytes(r->dtype);
  return {name, p, r->rows, r->vocab * es, stride * es, written, true};
}

// Refuses a call that writes into another of its arrays.
template <size_t N> int CheckApart(const char *fn, const mfh::Span (&spans)[N]) {
  size_t a = 0, b = 0;
  if (!mfh::FindOverlap(spans, &a, &b))
    return MFH_OK;
  return Invalid(fn, (std::string(spans[a].name) + " overlaps " + spans[b].name).c_str());
}

// No tensor on a card of 288 GB has more.
constexpr uint64_t kMostElements = uint64_t(1) << 38;

bool Finite(float v) { return std::isfinite(v); }

// Rows by themselves; on success `p` holds them.
int CheckRows(const char *fn, const mfh_policy_rows *r, mfh::RowLossParams *p) {
  if (r->rows < 0)
    return Invalid(fn, "rows must be >= 0");
  if (r->vocab < 1 || r->vocab > (1 << 30))
    return Invalid(fn, "vocab must be 1 .. 2^30");
  if (r->dtype < MFH_DTYPE_F32 || r->dtype > MFH_DTYPE_F16)
    return Invalid(fn, "unknown dtype");
  if (!(r->softmax_temp > 0.f) || !Finite(r->softmax_temp) || !Finite(1.f / r->softmax_temp))
    return Invalid(fn, "softmax_temp must be positive and finite");
  if (r->device < -1)
    return Invalid(fn, "device must be -1 or an ordinal");
  const std::int64_t most = INT64_MAX / 8;
  if (r->stride < r->vocab || (r->rows > 0 && r->stride > most / r->rows))
    return Invalid(fn, "stride must be at least vocab, and rows * stride addressable");
  if (r->n_moves < 0 || r->n_moves > INT32_MAX)
    return Invalid(fn, "n_moves must be 0 .. 2^31 - 1");
  if (!r->d_move_offsets && (r->d_move_indices || r->n_moves))
    return Invalid(fn, "move indices without offsets");
  if (r->d_move_offsets && r->n_moves > 0 && !r->d_move_indices)
    return Invalid(fn, "null move indices");
  if (r->d_move_offsets && r->vocab > 32768)
    return Invalid(fn, "move lists need vocab <= 32768");
  if (r->rows > 0 && !r->d_logits)
    return Invalid(fn, "null logits");
  if (!Aligned(r->d_logits, mfh::DTypeBytes(r->dtype)) || !Aligned(r->d_move_offsets, 4) ||
      !Aligned(r->d_move_indices, 2) || !Aligned(r->d_actions, 4))
    return Invalid(fn, "pointers must be aligned to their elements");
  p->x = r->d_logits;
  p->ldx = r->stride;
  p->rows = r->rows;
  p->vocab = r->vocab;
  p->dtype = r->dtype;
  p->offsets = r->d_move_offsets;
  p->indices = r->d_move_indices;
  p->n_moves = r->n_moves;
  p->actions = r->d_actions;
  p->inv_temp = 1.f / r->softmax_temp;
  return MFH_OK;
}

int CheckGrad(const char *fn, const mfh_policy_rows *r, void *grad, std::int64_t stride) {
  if (!grad)
    return MFH_OK;
  const int es = mfh::DTypeBytes(r->dtype);
  if (stride < r->vocab || (r->rows > 0 && stride > INT64_MAX / 8 / r->rows))
    return Invalid(fn, "grad_stride must be at least vocab, and rows * stride addressable");
  if (!Aligned(grad, es))
    return Invalid(fn, "pointers must be aligned to their elements");
  if (r->rows > 0 && mfh::RowsClash(r->d_logits, r->stride * es, grad, stride * es, r->rows,
                                    static_cast<std::int64_t>(r->vocab) * es))
    return Invalid(fn, "d_grad overlaps d_logits without being it");
  return MFH_OK;
}

}  // namespace

extern "C" {

int mfh_policy_loss_device(const mfh_policy_rows *rows, const mfh_policy_loss *loss,
                           void *stream) {
  const char *fn = "mfh_policy_loss_device";
  if (!rows || !loss)
    return Invalid(fn, "null argument");
  try {
    mfh::RowLossParams p;
    int rc = CheckRows(fn, rows, &p);
    if (rc != MFH_OK)
      return rc;
    const int es = mfh::DTypeBytes(rows->dtype);
    if (!(loss->clip_low >= 0.f) || !(loss->clip_high >= 0.f))
      return Invalid(fn, "clip_low and clip_high must be >= 0");
    if (!Finite(loss->kl_coef) || !Finite(loss->entropy_coef))
      return Invalid(fn, "kl_coef and entropy_coef must be finite");
    if (!loss->d_ref_logits && (loss->kl_coef != 0.f || loss->d_kl))
      return Invalid(fn, "kl_coef and d_kl need reference logits");
    if (loss->d_ref_logits &&
        (loss->ref_stride < rows->vocab ||
         (rows->rows > 0 && loss->ref_stride > INT64_MAX / 8 / rows->rows)))
      return Invalid(fn, "ref_stride must be at least vocab, and rows * stride addressable");
    if (!Aligned(loss->d_ref_logits, es) || !Aligned(loss->d_old_logp, 4) ||
        !Aligned(loss->d_advantage, 4) || !Aligned(loss->d_weight, 4) ||
        !Aligned(loss->d_loss, 4) || !Aligned(loss->d_logp, 4) || !Aligned(loss->d_kl, 4) ||
        !Aligned(loss->d_entropy, 4))
      return Invalid(fn, "pointers must be aligned to their elements");
    rc = CheckGrad(fn, rows, loss->d_grad, loss->grad_stride);
    if (rc != MFH_OK)
      return rc;
    if (rows->rows > 0 && loss->d_grad && loss->d_ref_logits &&
        mfh::RowsClash(loss->d_ref_logits, loss->ref_stride * es, loss->d_grad,
                       loss->grad_stride * es, rows->rows,
                       static_cast<std::int64_t>(rows->vocab) * es))
      return Invalid(fn, "d_grad overlaps d_ref_logits without being it");
    if (rows->rows == 0)
      return MFH_OK;
    OnDevice on;
    const Named ptrs[] = {{"d_logits", rows->d_logits},
                          {"d_move_offsets", rows->d_move_offsets},
                          {"d_move_indices", rows->d_move_indices},
                          {"d_actions", rows->d_actions},
                          {"d_old_logp", loss->d_old_logp},
                          {"d_advantage", loss->d_advantage},
                          {"d_weight", loss->d_weight},
                          {"d_ref_logits", loss->d_ref_logits},
                          {"d_loss", loss->d_loss},
                          {"d_logp", loss->d_logp},
                          {"d_kl", loss->d_kl},
                          {"d_entropy", loss->d_entropy},
                          {"d_grad", loss->d_grad}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, rows->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    const std::int64_t column = rows->rows * 4;
    const mfh::Span spans[] = {
        Rows("d_logits", rows->d_logits, rows, rows->stride, false),
        Flat("d_move_offsets", rows->d_move_offsets, column + 4, false),
        Flat("d_move_indices", rows->d_move_indices, rows->n_moves * 2, false),
        Flat("d_actions", rows->d_actions, column, false),
        Flat("d_old_logp", loss->d_old_logp, column, false),
        Flat("d_advantage", loss->d_advantage, column, false),
        Flat("d_weight", loss->d_weight, column, false),
        Rows("d_ref_logits", loss->d_ref_logits, rows, loss->ref_stride, false),
        Flat("d_loss", loss->d_loss, column, true),
        Flat("d_logp", loss->d_logp, column, true),
        Flat("d_kl", loss->d_kl, column, true),
        Flat("d_entropy", loss->d_entropy, column, true),
        Rows("d_grad", loss->d_grad, rows, loss->grad_stride, true)};
    rc = CheckApart(fn, spans);
    if (rc != MFH_OK)
      return rc;
    p.old_logp = loss->d_old_logp;
    p.advantage = loss->d_advantage;
    p.weight = loss->d_weight;
    if (loss->d_kl || loss->kl_coef != 0.f) {
      p.y = loss->d_ref_logits;
      p.ldy = loss->ref_stride;
    }
    p.ratio_low = 1.f - loss->clip_low;
    p.ratio_high = 1.f + loss->clip_high;
    p.kl_coef = loss->kl_coef;
    p.entropy_coef = loss->entropy_coef;
    p.loss = loss->d_loss;
    p.logp = loss->d_logp;
    p.kl = loss->d_kl;
    p.entropy = loss->d_entropy;
    p.g = loss->d_grad;
    p.ldg = loss->grad_stride;
    std::string err;
    const hipError_t e = mfh::LaunchRowLoss(p, st, &err);
    return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_preference_loss_workspace_bytes(int64_t rows, uint64_t *bytes) {
  if (!bytes || rows < 0 || rows > INT64_MAX / 16)
    return Invalid("mfh_preference_loss_workspace_bytes", "bad arguments");
  *bytes = 2 * sizeof(float) * static_cast<uint64_t>(rows);
  return MFH_OK;
}

int mfh_preference_loss_device(const mfh_policy_rows *rows, const mfh_preference_loss *loss,
                               void *stream) {
  const char *fn = "mfh_preference_loss_device";
  if (!rows || !loss)
    return Invalid(fn, "null argument");
  try {
    mfh::RowLossParams p;
    int rc = CheckRows(fn, rows, &p);
    if (rc != MFH_OK)
      return rc;
    if (loss->pairs < 0 || loss->pairs > (1 << 23))
      return Invalid(fn, "pairs must be 0 .. 2^23");
    if (loss->kind < MFH_PREFERENCE_SIGMOID || loss->kind > MFH_PREFERENCE_SQUARE)
      return Invalid(fn, "unknown kind");
    if (!(loss->beta > 0.f) || !Finite(loss->beta))
      return Invalid(fn, "beta must be positive and finite");
    if (!(loss->label_smoothing >= 0.f && loss->label_smoothing <= 0.5f) ||
        (loss->kind != MFH_PREFERENCE_SIGMOID && loss->label_smoothing != 0.f))
      return Invalid(fn, "label_smoothing must be 0 .. 0.5, and 0 but for the sigmoid loss");
    if (loss->average != 0 && loss->average != 1)
      return Invalid(fn, "average must be 0 or 1");
    if (loss->pairs > 0 && !loss->d_seq_offsets)
      return Invalid(fn, "null sequence offsets");
    if (!Aligned(loss->d_seq_offsets, 4) || !Aligned(loss->d_ref_logp, 4) ||
        !Aligned(loss->d_weight, 4) || !Aligned(loss->d_loss, 4) || !Aligned(loss->d_margin, 4) ||
        !Aligned(loss->d_logp, 4) || !Aligned(loss->d_workspace, 8))
      return Invalid(fn, "pointers must be aligned to their elements");
    rc = CheckGrad(fn, rows, loss->d_grad, loss->grad_stride);
    if (rc != MFH_OK)
      return rc;
    uint64_t need = 0;
    rc = mfh_preference_loss_workspace_bytes(rows->rows, &need);
    if (rc != MFH_OK)
      return rc;
    if (need > 0 && (!loss->d_workspace || loss->workspace_bytes < need))
      return Invalid(fn, "the workspace is too small");
    if (loss->pairs == 0)
      return MFH_OK;
    OnDevice on;
    const Named ptrs[] = {{"d_logits", rows->d_logits},
                          {"d_seq_offsets", loss->d_seq_offsets},
                          {"d_move_offsets", rows->d_move_offsets},
                          {"d_move_indices", rows->d_move_indices},
                          {"d_actions", rows->d_actions},
                          {"d_ref_logp", loss->d_ref_logp},
                          {"d_weight", loss->d_weight},
                          {"d_loss", loss->d_loss},
                          {"d_margin", loss->d_margin},
                          {"d_logp", loss->d_logp},
                          {"d_grad", loss->d_grad},
                          {"d_workspace", need > 0 ? loss->d_workspace : nullptr}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, rows->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    const std::int64_t column = rows->rows * 4, pairs = loss->pairs * 4;
    const mfh::Span spans[] = {
        Rows("d_logits", rows->d_logits, rows, rows->stride, false),
        Flat("d_seq_offsets", loss->d_seq_offsets, 2 * pairs + 4, false),
        Flat("d_move_offsets", rows->d_move_offsets, column + 4, false),
        Flat("d_move_indices", rows->d_move_indices, rows->n_moves * 2, false),
        Flat("d_actions", rows->d_actions, column, false),
        Flat("d_ref_logp", loss->d_ref_logp, column, false),
        Flat("d_weight", loss->d_weight, pairs, false),
        Flat("d_loss", loss->d_loss, pairs, true),
        Flat("d_margin", loss->d_margin, pairs, true),
        Flat("d_logp", loss->d_logp, column, true),
        Flat("d_workspace", need > 0 ? loss->d_workspace : nullptr,
             static_cast<std::int64_t>(need), true),
        Rows("d_grad", loss->d_grad, rows, loss->grad_stride, true)};
    rc = CheckApart(fn, spans);
    if (rc != MFH_OK)
      return rc;
    p.g = loss->d_grad;
    p.ldg = loss->grad_stride;
    mfh::PairLossParams q;
    q.seq_offsets = loss->d_seq_offsets;
    q.pairs = loss->pairs;
    q.rows = rows->rows;
    q.mark = static_cast<float *>(loss->d_workspace);
    q.coef = q.mark + rows->rows;
    q.ref_logp = loss->d_ref_logp;
    q.weight = loss->d_weight;
    q.kind = loss->kind;
    q.average = loss->average != 0;
    q.beta = loss->beta;
    q.smoothing = loss->label_smoothing;
    q.loss = loss->d_loss;
    q.margin = loss->d_margin;
    q.logp = loss->d_logp;
    std::string err;
    const hipError_t e = mfh::LaunchPreference(p, q, st, &err);
    return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_grad_set_create(const mfh_grad_tensor *tensors, int n_tensors, int device,
                        mfh_grad_set **out) {
  const char *fn = "mfh_grad_set_create";
  if (!out || n_tensors < 0 || (n_tensors > 0 && !tensors) || device < -1)
    return Invalid(fn, "bad arguments");
  *out = nullptr;
  try {
    // Every byte range that is written, and every one that is read.
    struct Range {
      std::uintptr_t begin, end;
      int tensor;
      bool written;
    };
    std::vector<Range> ranges;
    for (int i = 0; i < n_tensors; ++i) {
      const mfh_grad_tensor &t = tensors[i];
      if (t.dtype < MFH_DTYPE_F32 || t.dtype > MFH_DTYPE_F16)
        return Invalid(fn, "unknown dtype");
      if (t.count == 0)
        continue;
      const int es = mfh::DTypeBytes(t.dtype);
      if (!t.src || t.count > kMostElements)
        return Invalid(fn, "a tensor without memory, or too large");
      if (!Aligned(t.src, es) || !Aligned(t.dst, es))
        return Invalid(fn, "pointers must be aligned to their elements");
      const auto add = [&](const void *p, bool written) {
        const auto b = reinterpret_cast<std::uintptr_t>(p);
        ranges.push_back({b, b + static_cast<std::uintptr_t>(t.count) * es, i, written});
      };
      add(t.src, false);
      if (t.dst)
        add(t.dst, true);
    }
    // In order of their beginning, a range meets an earlier one exactly when
    // it begins before the furthest end so far, of those written or (if it
    // is written itself) of any.
    std::sort(ranges.begin(), ranges.end(),
              [](const Range &a, const Range &b) { return a.begin < b.begin; });
    std::vector<Range> open;
    for (const Range &r : ranges) {
      open.erase(std::remove_if(open.begin(), open.end(),
                                [&](const Range &o) { return o.end <= r.begin; }),
                 open.end());
      for (const Range &o : open) {
        const bool itself = o.tensor == r.tensor && o.written != r.written &&
                            o.begin == r.begin && o.end == r.end;
        if ((o.written || r.written) && !itself)
          return Invalid(fn, "a dst overlaps another tensor, or its own src in part");
      }
      open.push_back(r);
    }

    int rc = NeedDevice(fn, device);
    if (rc != MFH_OK)
      return rc;
    int dev = device;
    for (int i = 0; i < n_tensors; ++i) {
      if (tensors[i].count == 0)
        continue;
      rc = PointerDevice(fn, "src", tensors[i].src, dev, &dev);
      if (rc == MFH_OK && tensors[i].dst)
        rc = PointerDevice(fn, "dst", tensors[i].dst, dev, nullptr);
      if (rc != MFH_OK)
        return rc;
    }
    if (dev < 0) {
      const hipError_t e = hipGetDevice(&dev);
      if (e != hipSuccess)
        return HipError(fn, "hipGetDevice", e);
    }
    if (!IsGfx950(dev))
      return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": the device is not gfx950 (MI355X)");
    OnDevice on;
    hipError_t e = on.Set(dev);
    if (e != hipSuccess)
      return HipError(fn, "hipSetDevice", e);
    std::vector<mfh::ByteRange> memory;
    for (const Range &r : ranges)
      memory.push_back({r.begin, r.end});
    std::vector<mfh::GradChunk> chunks;
    for (int i = 0; i < n_tensors; ++i) {
      const mfh_grad_tensor &t = tensors[i];
      const int es = mfh::DTypeBytes(t.dtype);
      const uint64_t most = mfh::kGradChunkBytes / es;
      for (uint64_t at = 0; at < t.count; at += most) {
        const uint64_t n = std::min<uint64_t>(most, t.count - at);
        chunks.push_back({static_cast<const char *>(t.src) + at * es,
                          t.dst ? static_cast<char *>(t.dst) + at * es : nullptr,
                          static_cast<std::int32_t>(n), t.dtype});
      }
    }
    auto set = std::make_unique<mfh_grad_set>();
    set->device = dev;
    set->memory = mfh::Joined(std::move(memory));
    set->n_chunks = static_cast<std::int64_t>(chunks.size());
    std::int64_t total = 0;
    for (const mfh::GradChunk &c : chunks)
      total += static_cast<std::int64_t>(c.count) * mfh::DTypeBytes(c.dtype);
    set->past = total > mfh::kGradCachedBytes;
    if (!chunks.empty()) {
      const size_t bytes = chunks.size() * sizeof(mfh::GradChunk);
      e = hipMalloc(reinterpret_cast<void **>(&set->chunks), bytes);
      if (e != hipSuccess) {
        (void)hipGetLastError();
        return SetError(MFH_ERR_OUT_OF_MEMORY, std::string(fn) + ": chunk list allocation failed");
      }
      e = hipMemcpy(set->chunks, chunks.data(), bytes, hipMemcpyHostToDevice);
      if (e != hipSuccess) {
        (void)hipFree(set->chunks);
        return HipError(fn, "hipMemcpy", e);
      }
    }
    *out = set.release();
    return MFH_OK;
  } catch (const std::bad_alloc &) {
    return SetError(MFH_ERR_OUT_OF_MEMORY, std::string(fn) + ": out of host memory");
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

void mfh_grad_set_destroy(mfh_grad_set *set) {
  if (!set)
    return;
  OnDevice on;
  (void)on.Set(set->device);
  if (set->chunks)
    (void)hipFree(set->chunks);
  delete set;
}

int mfh_grad_workspace_bytes(const mfh_grad_set *set, uint64_t *bytes) {
  if (!set || !bytes)
    return Invalid("mfh_grad_workspace_bytes", "null argument");
  *bytes = sizeof(double) * static_cast<uint64_t>(mfh::GradNormGroups(set->n_chunks));
  return MFH_OK;
}

int mfh_grad_norm_device(const mfh_grad_set *set, double *d_sumsq, void *d_workspace,
                         uint64_t workspace_bytes, void *stream) {
  const char *fn = "mfh_grad_norm_device";
  if (!set || !d_sumsq || !d_workspace)
    return Invalid(fn, "null argument");
  const int groups = mfh::GradNormGroups(set->n_chunks);
  if (workspace_bytes < sizeof(double) * static_cast<uint64_t>(groups))
    return Invalid(fn, "the workspace is too small");
  if (!Aligned(d_sumsq, 8) || !Aligned(d_workspace, 8))
    return Invalid(fn, "pointers must be aligned to their elements");
  if (mfh::Meets(set->memory, d_sumsq, sizeof(double)) ||
      mfh::Meets(set->memory, d_workspace, sizeof(double) * static_cast<uint64_t>(groups)))
    return Invalid(fn, "d_sumsq or the workspace lies in a gradient");
  try {
    OnDevice on;
    const Named ptrs[] = {{"d_sumsq", d_sumsq}, {"d_workspace", d_workspace}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = Enter(fn, set->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    std::string err;
    double *partials = static_cast<double *>(d_workspace);
    hipError_t e = mfh::LaunchGradSumsq(set->chunks, set->n_chunks, set->past, partials, st, &err);
    if (e == hipSuccess)
      e = mfh::LaunchGradSum(partials, groups, d_sumsq, st, &err);
    return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_grad_scale_device(const mfh_grad_set *set, const double *d_sumsq, float max_norm,
                          void *stream) {
  const char *fn = "mfh_grad_scale_device";
  if (!set || !d_sumsq)
    return Invalid(fn, "null argument");
  if (!(max_norm >= 0.f))
    return Invalid(fn, "max_norm must be >= 0");
  if (!Aligned(d_sumsq, 8))
    return Invalid(fn, "pointers must be aligned to their elements");
  if (mfh::Meets(set->memory, d_sumsq, sizeof(double)))
    return Invalid(fn, "d_sumsq lies in a gradient");
  try {
    OnDevice on;
    const Named ptrs[] = {{"d_sumsq", d_sumsq}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = Enter(fn, set->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    std::string err;
    const hipError_t e = mfh::LaunchGradScale(set->chunks, set->n_chunks, set->past, d_sumsq,
                                              1, max_norm, nullptr, st, &err);
    return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_grad_clip_device(const mfh_grad_set *set, float max_norm, float *d_norm,
                         void *d_workspace, uint64_t workspace_bytes, void *stream) {
  const char *fn = "mfh_grad_clip_device";
  if (!set || !d_workspace)
    return Invalid(fn, "null argument");
  if (!(max_norm >= 0.f))
    return Invalid(fn, "max_norm must be >= 0");
  const int groups = mfh::GradNormGroups(set->n_chunks);
  if (workspace_bytes < sizeof(double) * static_cast<uint64_t>(groups))
    return Invalid(fn, "the workspace is too small");
  if (!Aligned(d_norm, 4) || !Aligned(d_workspace, 8))
    return Invalid(fn, "pointers must be aligned to their elements");
  // One workgroup writes the norm while others still sum the workspace.
  const auto norm = reinterpret_cast<std::uintptr_t>(d_norm),
             work = reinterpret_cast<std::uintptr_t>(d_workspace);
  if (d_norm && norm < work + sizeof(double) * groups && work < norm + sizeof(float))
    return Invalid(fn, "d_norm lies in the workspace");
  if ((d_norm && mfh::Meets(set->memory, d_norm, sizeof(float))) ||
      mfh::Meets(set->memory, d_workspace, sizeof(double) * static_cast<uint64_t>(groups)))
    return Invalid(fn, "d_norm or the workspace lies in a gradient");
  try {
    OnDevice on;
    const Named ptrs[] = {{"d_workspace", d_workspace}, {"d_norm", d_norm}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = Enter(fn, set->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    std::string err;
    double *partials = static_cast<double *>(d_workspace);
    hipError_t e = mfh::LaunchGradSumsq(set->chunks, set->n_chunks, set->past, partials, st, &err);
    if (e == hipSuccess)
      e = mfh::LaunchGradScale(set->chunks, set->n_chunks, set->past, partials, groups,
                               max_norm, d_norm, st, &err);
    return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

}  // extern "C"
