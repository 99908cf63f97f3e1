// C ABI of the layers of a training step (include/mfhip.h): layer norm,
// attention, AdamW.  Argument checks, the device and stream of a call, and the
// launches.  Shapes are checked before any device is touched.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <memory>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/mfhip.h"
#include "learn_checks.h"
#include "learn_ranges.h"
#include "mfh_kernels.h"
#include "mfh_status.h"

struct mfh_adamw_set {
  int device = 0;
  std::int64_t n_chunks = 0;
  bool eight = false;
  bool past = false;               // too large for the caches
  mfh::AdamChunk *chunks = nullptr;  // device memory, read only
  std::vector<mfh::ByteRange> memory;
};

using namespace mfh::checks;

namespace {

// No array on a card of 288 GB reaches further.
constexpr std::int64_t kMostBytes = std::int64_t(1) << 40;

bool KnownType(int dtype) { return dtype >= MFH_DTYPE_F32 && dtype <= MFH_DTYPE_F16; }

int CheckApart(const char *fn, const std::vector<mfh::Region> &regions) {
  for (size_t i = 0; i < regions.size(); ++i)
    for (size_t j = 0; j < i; ++j) {
      const mfh::Region &x = regions[i], &y = regions[j];
      if ((x.written || y.written) && !mfh::Apart(x, y))
        return Invalid(fn, (std::string(x.written ? x.name : y.name) + " overlaps " +
                            (x.written ? y.name : x.name))
                               .c_str());
    }
  return MFH_OK;
}

// ---- Layer norm ----

int CheckNorm(const char *fn, const mfh_norm_rows *r, mfh::NormParams *p) {
  if (r->rows < 0)
    return Invalid(fn, "rows must be >= 0");
  if (r->width < 1 || r->width > (1 << 20))
    return Invalid(fn, "width must be 1 .. 2^20");
  if (!KnownType(r->dtype))
    return Invalid(fn, "unknown dtype");
  if (!Finite(r->alpha))
    return Invalid(fn, "alpha must be finite");
  if (!(r->eps >= 0.f) || !Finite(r->eps))
    return Invalid(fn, "eps must be finite and >= 0");
  if (r->device < -1)
    return Invalid(fn, "device must be -1 or an ordinal");
  if (r->rows > 0 && !r->d_x)
    return Invalid(fn, "null x");
  if (!Aligned(r->d_gamma, 4) || !Aligned(r->d_beta, 4))
    return Invalid(fn, "pointers must be aligned to their elements");
  p->rows = r->rows;
  p->width = r->width;
  p->dtype = r->dtype;
  p->alpha = r->alpha;
  p->eps = r->eps;
  p->gamma = r->d_gamma;
  p->beta = r->d_beta;
  return MFH_OK;
}

// Rows of one array of a call: its stride, and where it lies.
int CheckRowArray(const char *fn, const mfh_norm_rows *r, const char *name, const void *ptr,
                  std::int64_t stride, bool written, std::vector<mfh::Region> *regions) {
  if (!ptr)
    return MFH_OK;
  const std::int64_t es = mfh::DTypeBytes(r->dtype);
  if (stride < r->width || (r->rows > 0 && stride > kMostBytes / es / r->rows))
    return Invalid(fn, (std::string(name) + ": the stride must be at least the width, and rows * "
                                            "stride addressable")
                           .c_str());
  if (!Aligned(ptr, es))
    return Invalid(fn, "pointers must be aligned to their elements");
  regions->push_back(mfh::RegionOf(name, ptr, r->width * es, written, {{r->rows, stride * es}}));
  return MFH_OK;
}

// Arrays of a call apart from each other, but for an output that is one of
// the inputs, row for row.
int CheckNormApart(const char *fn, const std::vector<mfh::Region> &regions) {
  for (size_t i = 0; i < regions.size(); ++i)
    for (size_t j = 0; j < i; ++j) {
      const mfh::Region &x = regions[i], &y = regions[j];
      if (!(x.written || y.written) || mfh::Apart(x, y))
        continue;
      const bool in_place = x.written != y.written && x.inner == y.inner && x.p == y.p &&
                            x.dims[0].n == y.dims[0].n && x.dims[0].stride > 0 &&
                            x.dims[0].stride == y.dims[0].stride;
      if (!in_place)
        return Invalid(fn, (std::string(x.written ? x.name : y.name) + " overlaps " +
                            (x.written ? y.name : x.name))
                               .c_str());
    }
  return MFH_OK;
}

void AddFlat(const char *name, const void *p, std::int64_t bytes, bool written,
             std::vector<mfh::Region> *regions) {
  if (p && bytes > 0)
    regions->push_back(mfh::RegionOf(name, p, bytes, written, {}));
}

// ---- Attention ----

int CheckHeads(const char *fn, const char *name, const mfh_attention *a, const mfh_heads &v,
               int heads, int tokens, bool written, std::vector<mfh::Region> *regions,
               mfh::HeadsView *out) {
  const std::int64_t es = mfh::DTypeBytes(a->dtype);
  const auto bad = [&](const char *what) {
    return Invalid(fn, (std::string(name) + ": " + what).c_str());
  };
  const std::int64_t n[3] = {a->batch, tokens, heads}, stride[3] = {v.batch, v.token, v.head};
  std::int64_t reach = a->dim;
  for (int i = 0; i < 3; ++i) {
    if (stride[i] < 0 || (n[i] > 1 && stride[i] > kMostBytes / (n[i] - 1)))
      return bad("strides must be >= 0 and the array addressable");
    if (n[i] > 1)
      reach += (n[i] - 1) * stride[i];
  }
  if (n[1] > 1 && stride[1] > INT64_C(0xFFFFFFFF))
    return bad("strides of tokens must be below 2^32");
  if (reach > kMostBytes / es)
    return bad("strides must be >= 0 and the array addressable");
  if (n[0] == 0 || n[1] == 0)
    return MFH_OK;  // nothing in it
  if (!v.p)
    return bad("null array");
  if (!Aligned(v.p, es))
    return Invalid(fn, "pointers must be aligned to their elements");
  const mfh::Region r = mfh::RegionOf(name, v.p, a->dim * es, written,
                                      {{n[0], n[0] > 1 ? stride[0] * es : 0},
                                       {n[1], n[1] > 1 ? stride[1] * es : 0},
                                       {n[2], n[2] > 1 ? stride[2] * es : 0}});
  if (written && !mfh::Nested(r))
    return bad("a written array has no two elements in one place");
  regions->push_back(r);
  *out = {v.p, v.batch, v.token, v.head};
  return MFH_OK;
}

int CheckAttention(const char *fn, const mfh_attention *a, std::vector<mfh::Region> *regions,
                   mfh::TrainAttention *t) {
  if (a->batch < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
    return Invalid(fn, "batch must be >= 0, heads a multiple of kv_heads, both >= 1");
  if (a->q_len < 0 || a->k_len < 0 || a->k_len > (1 << 30))
    return Invalid(fn, "q_len and k_len must be 0 .. 2^30");
  const std::int64_t group = a->heads / a->kv_heads;
  if (a->q_len * group > (1 << 30) || static_cast<std::int64_t>(a->batch) * a->heads > (1 << 30))
    return Invalid(fn, "q_len * heads / kv_heads and batch * heads must be at most 2^30");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8 != 0)
    return Invalid(fn, "dim must be a multiple of 8, 8 .. 128");
  if (!KnownType(a->dtype) || (a->d_bias && !KnownType(a->bias_dtype)))
    return Invalid(fn, "unknown dtype");
  if (a->causal != 0 && a->causal != 1)
    return Invalid(fn, "causal must be 0 or 1");
  if (!Finite(a->scale))
    return Invalid(fn, "scale must be finite");
  if (a->device < -1)
    return Invalid(fn, "device must be -1 or an ordinal");
  if (!Aligned(a->d_q_lengths, 4) || !Aligned(a->d_k_lengths, 4))
    return Invalid(fn, "pointers must be aligned to their elements");
  t->batch = a->batch;
  t->heads = a->heads;
  t->kv_heads = a->kv_heads;
  t->group = static_cast<int>(group);
  t->q_len = a->q_len;
  t->k_len = a->k_len;
  t->dim = a->dim;
  t->dtype = a->dtype;
  t->scale = a->scale;
  t->causal = a->causal != 0;
  t->bias = a->d_bias;
  t->q_lengths = a->d_q_lengths;
  t->k_lengths = a->d_k_lengths;
  int rc = CheckHeads(fn, "q", a, a->q, a->heads, a->q_len, false, regions, &t->q);
  if (rc == MFH_OK)
    rc = CheckHeads(fn, "k", a, a->k, a->kv_heads, a->k_len, false, regions, &t->k);
  if (rc == MFH_OK)
    rc = CheckHeads(fn, "v", a, a->v, a->kv_heads, a->k_len, false, regions, &t->v);
  if (rc != MFH_OK)
    return rc;
  AddFlat("d_q_lengths", a->d_q_lengths, 4 * std::int64_t(a->batch), false, regions);
  AddFlat("d_k_lengths", a->d_k_lengths, 4 * std::int64_t(a->batch), false, regions);
  return MFH_OK;
}

// The bias (or, laid out alike, its gradient), one of each of its planes.
int CheckBias(const char *fn, const char *name, const mfh_attention *a, const void *ptr,
              bool written, std::vector<mfh::Region> *regions) {
  if (!ptr || a->batch == 0 || a->q_len == 0 || a->k_len == 0)
    return MFH_OK;
  const std::int64_t es = mfh::DTypeBytes(a->bias_dtype);
  const std::int64_t stride[3] = {a->bias_batch, a->bias_head, a->bias_query};
  const std::int64_t n[3] = {a->batch, a->heads, a->q_len};
  std::vector<mfh::Region::Dim> dims;
  std::int64_t reach = a->k_len;
  for (int i = 0; i < 3; ++i) {
    if (stride[i] < 0 || (n[i] > 1 && stride[i] > kMostBytes / (n[i] - 1)))
      return Invalid(fn, "bias strides must be >= 0 and the bias addressable");
    if (n[i] > 1)
      reach += (n[i] - 1) * stride[i];
    dims.push_back({stride[i] ? n[i] : 1, n[i] > 1 ? stride[i] * es : 0});
  }
  if (reach > kMostBytes / es)
    return Invalid(fn, "bias strides must be >= 0 and the bias addressable");
  if (!Aligned(ptr, es))
    return Invalid(fn, "pointers must be aligned to their elements");
  const mfh::Region r = mfh::RegionOf(name, ptr, a->k_len * es, written, dims);
  if (written && (!mfh::Nested(r) || (a->bias_query == 0 && a->q_len > 1)))
    return Invalid(fn, "d_dbias: a gradient for each query, and no two elements in one place");
  regions->push_back(r);
  return MFH_OK;
}

int NeedWorkspace(const char *fn, const void *p, uint64_t bytes, uint64_t need) {
  if (need > 0 && (!p || bytes < need))
    return Invalid(fn, "the workspace is too small");
  if (!Aligned(p, 16))
    return Invalid(fn, "the workspace must be 16-byte aligned");
  return MFH_OK;
}

int Done(const char *fn, hipError_t e, const std::string &err) {
  return e == hipSuccess ? MFH_OK : HipError(fn, err.empty() ? "launch" : err.c_str(), e);
}

}  // namespace

extern "C" {

int mfh_layer_norm_device(const mfh_norm_rows *rows, void *d_y, int64_t y_stride, float *d_mean,
                          float *d_rstd, void *stream) {
  const char *fn = "mfh_layer_norm_device";
  if (!rows)
    return Invalid(fn, "null argument");
  try {
    mfh::NormParams p;
    int rc = CheckNorm(fn, rows, &p);
    std::vector<mfh::Region> regions;
    if (rc == MFH_OK)
      rc = CheckRowArray(fn, rows, "d_x", rows->d_x, rows->x_stride, false, &regions);
    if (rc == MFH_OK)
      rc = CheckRowArray(fn, rows, "d_residual", rows->d_residual, rows->residual_stride, false,
                         &regions);
    if (rc == MFH_OK)
      rc = CheckRowArray(fn, rows, "d_y", d_y, y_stride, true, &regions);
    if (rc != MFH_OK)
      return rc;
    if (!Aligned(d_mean, 4) || !Aligned(d_rstd, 4))
      return Invalid(fn, "pointers must be aligned to their elements");
    if (rows->rows == 0)
      return MFH_OK;
    const std::int64_t column = 4 * rows->rows, weights = 4 * std::int64_t(rows->width);
    AddFlat("d_gamma", rows->d_gamma, weights, false, &regions);
    AddFlat("d_beta", rows->d_beta, weights, false, &regions);
    AddFlat("d_mean", d_mean, column, true, &regions);
    AddFlat("d_rstd", d_rstd, column, true, &regions);
    rc = CheckNormApart(fn, regions);
    if (rc != MFH_OK)
      return rc;
    OnDevice on;
    const Named ptrs[] = {{"d_x", rows->d_x},       {"d_residual", rows->d_residual},
                          {"d_gamma", rows->d_gamma}, {"d_beta", rows->d_beta},
                          {"d_y", d_y},             {"d_mean", d_mean},
                          {"d_rstd", d_rstd}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, rows->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    p.x = rows->d_x;
    p.ldx = rows->x_stride;
    p.residual = rows->d_residual;
    p.ldr = rows->residual_stride;
    p.y = d_y;
    p.ldy = y_stride;
    p.mean = d_mean;
    p.rstd = d_rstd;
    std::string err;
    const hipError_t e = mfh::LaunchNorm(p, st, &err);
    return Done(fn, e, err);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_layer_norm_workspace_bytes(int64_t rows, int32_t width, uint64_t *bytes) {
  if (!bytes || rows < 0 || width < 1 || width > (1 << 20))
    return Invalid("mfh_layer_norm_workspace_bytes", "bad arguments");
  *bytes = 8ull * static_cast<uint64_t>(width) *
           static_cast<uint64_t>(mfh::NormPartials(rows, width));
  return MFH_OK;
}

int mfh_layer_norm_backward_device(const mfh_norm_rows *rows, const mfh_norm_grads *grads,
                                   void *stream) {
  const char *fn = "mfh_layer_norm_backward_device";
  if (!rows || !grads)
    return Invalid(fn, "null argument");
  try {
    mfh::NormParams p;
    int rc = CheckNorm(fn, rows, &p);
    if (rc == MFH_OK && rows->rows > 0 && (!grads->d_dy || !grads->d_mean || !grads->d_rstd))
      rc = Invalid(fn, "null dy, mean or rstd");
    if (rc == MFH_OK && grads->d_dresidual && !rows->d_residual)
      rc = Invalid(fn, "d_dresidual without a residual");
    std::vector<mfh::Region> regions;
    const struct {
      const char *name;
      const void *p;
      std::int64_t stride;
      bool written;
    } arrays[] = {{"d_x", rows->d_x, rows->x_stride, false},
                  {"d_residual", rows->d_residual, rows->residual_stride, false},
                  {"d_dy", grads->d_dy, grads->dy_stride, false},
                  {"d_dx", grads->d_dx, grads->dx_stride, true},
                  {"d_dresidual", grads->d_dresidual, grads->dresidual_stride, true}};
    for (const auto &x : arrays)
      if (rc == MFH_OK)
        rc = CheckRowArray(fn, rows, x.name, x.p, x.stride, x.written, &regions);
    if (rc != MFH_OK)
      return rc;
    if (!Aligned(grads->d_mean, 4) || !Aligned(grads->d_rstd, 4) || !Aligned(grads->d_dgamma, 4) ||
        !Aligned(grads->d_dbeta, 4) || !Aligned(grads->d_workspace, 4))
      return Invalid(fn, "pointers must be aligned to their elements");
    const bool sums = grads->d_dgamma || grads->d_dbeta;
    uint64_t need = 0;
    rc = mfh_layer_norm_workspace_bytes(rows->rows, rows->width, &need);
    if (rc != MFH_OK)
      return rc;
    if (!sums)
      need = 0;
    if (need > 0 && (!grads->d_workspace || grads->workspace_bytes < need))
      return Invalid(fn, "the workspace is too small");
    if (!sums && (rows->rows == 0 || (!grads->d_dx && !grads->d_dresidual)))
      return MFH_OK;
    const void *workspace = need > 0 ? grads->d_workspace : nullptr;
    const std::int64_t column = 4 * rows->rows, weights = 4 * std::int64_t(rows->width);
    AddFlat("d_gamma", rows->d_gamma, weights, false, &regions);
    AddFlat("d_mean", grads->d_mean, column, false, &regions);
    AddFlat("d_rstd", grads->d_rstd, column, false, &regions);
    AddFlat("d_dgamma", grads->d_dgamma, weights, true, &regions);
    AddFlat("d_dbeta", grads->d_dbeta, weights, true, &regions);
    AddFlat("d_workspace", workspace, static_cast<std::int64_t>(need), true, &regions);
    rc = CheckNormApart(fn, regions);
    if (rc != MFH_OK)
      return rc;
    OnDevice on;
    const bool any = rows->rows > 0;
    const Named ptrs[] = {{"d_x", any ? rows->d_x : nullptr},
                          {"d_residual", any ? rows->d_residual : nullptr},
                          {"d_gamma", rows->d_gamma},
                          {"d_dy", any ? grads->d_dy : nullptr},
                          {"d_mean", any ? grads->d_mean : nullptr},
                          {"d_rstd", any ? grads->d_rstd : nullptr},
                          {"d_dx", any ? grads->d_dx : nullptr},
                          {"d_dresidual", any ? grads->d_dresidual : nullptr},
                          {"d_dgamma", grads->d_dgamma},
                          {"d_dbeta", grads->d_dbeta},
                          {"d_workspace", workspace}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, rows->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    p.x = rows->d_x;
    p.ldx = rows->x_stride;
    p.residual = rows->d_residual;
    p.ldr = rows->residual_stride;
    p.mean = const_cast<float *>(grads->d_mean);
    p.rstd = const_cast<float *>(grads->d_rstd);
    p.dy = grads->d_dy;
    p.lddy = grads->dy_stride;
    p.dx = grads->d_dx;
    p.lddx = grads->dx_stride;
    p.dresidual = grads->d_dresidual;
    p.lddr = grads->dresidual_stride;
    p.dgamma = grads->d_dgamma;
    p.dbeta = grads->d_dbeta;
    p.partials = need > 0 ? static_cast<float *>(grads->d_workspace) : nullptr;
    std::string err;
    const hipError_t e = mfh::LaunchNormBackward(p, st, &err);
    return Done(fn, e, err);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_attention_forward_workspace_bytes(const mfh_attention *a, uint64_t *bytes) {
  const char *fn = "mfh_attention_forward_workspace_bytes";
  if (!a || !bytes)
    return Invalid(fn, "null argument");
  try {
    mfh::TrainAttention t;
    std::vector<mfh::Region> regions;
    const int rc = CheckAttention(fn, a, &regions, &t);
    if (rc == MFH_OK)
      *bytes = mfh::AttentionForwardWorkspace(t);
    return rc;
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_attention_forward_device(const mfh_attention *a, const mfh_heads *out, float *d_lse,
                                 void *d_workspace, uint64_t workspace_bytes, void *stream) {
  const char *fn = "mfh_attention_forward_device";
  if (!a || !out)
    return Invalid(fn, "null argument");
  try {
    mfh::TrainAttention t;
    std::vector<mfh::Region> regions;
    int rc = CheckAttention(fn, a, &regions, &t);
    if (rc == MFH_OK)
      rc = CheckBias(fn, "d_bias", a, a->d_bias, false, &regions);
    if (rc == MFH_OK)
      rc = CheckHeads(fn, "out", a, *out, a->heads, a->q_len, true, &regions, &t.out);
    if (rc != MFH_OK)
      return rc;
    if (!Aligned(d_lse, 4))
      return Invalid(fn, "pointers must be aligned to their elements");
    const uint64_t need = mfh::AttentionForwardWorkspace(t);
    rc = NeedWorkspace(fn, d_workspace, workspace_bytes, need);
    if (rc != MFH_OK)
      return rc;
    if (a->batch == 0 || a->q_len == 0)
      return MFH_OK;
    void *workspace = need > 0 ? d_workspace : nullptr;
    AddFlat("d_lse", d_lse, 4 * std::int64_t(a->batch) * a->heads * a->q_len, true, &regions);
    AddFlat("d_workspace", workspace, static_cast<std::int64_t>(need), true, &regions);
    rc = CheckApart(fn, regions);
    if (rc != MFH_OK)
      return rc;
    OnDevice on;
    const bool keys = a->k_len > 0;
    const Named ptrs[] = {{"q", t.q.p},
                          {"k", t.k.p},
                          {"v", t.v.p},
                          {"out", t.out.p},
                          {"d_bias", keys ? a->d_bias : nullptr},
                          {"d_q_lengths", a->d_q_lengths},
                          {"d_k_lengths", a->d_k_lengths},
                          {"d_lse", d_lse},
                          {"d_workspace", workspace}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, a->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    t.bias_dtype = a->bias_dtype;
    t.bias_batch = a->bias_batch;
    t.bias_head = a->bias_head;
    t.bias_query = a->bias_query;
    t.lse = d_lse;
    t.workspace = workspace;
    std::string err;
    const hipError_t e = mfh::LaunchAttentionForward(t, st, &err);
    return Done(fn, e, err);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_attention_backward_workspace_bytes(const mfh_attention *a, uint64_t *bytes) {
  const char *fn = "mfh_attention_backward_workspace_bytes";
  if (!a || !bytes)
    return Invalid(fn, "null argument");
  try {
    mfh::TrainAttention t;
    std::vector<mfh::Region> regions;
    const int rc = CheckAttention(fn, a, &regions, &t);
    if (rc == MFH_OK)
      *bytes = mfh::AttentionBackwardWorkspace(t);
    return rc;
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_attention_backward_device(const mfh_attention *a, const mfh_attention_grads *grads,
                                  void *stream) {
  const char *fn = "mfh_attention_backward_device";
  if (!a || !grads)
    return Invalid(fn, "null argument");
  try {
    mfh::TrainAttention t;
    std::vector<mfh::Region> regions;
    int rc = CheckAttention(fn, a, &regions, &t);
    if (rc == MFH_OK)
      rc = CheckBias(fn, "d_bias", a, a->d_bias, false, &regions);
    if (rc == MFH_OK && grads->d_dbias && !a->d_bias)
      rc = Invalid(fn, "d_dbias without a bias");
    if (rc == MFH_OK)
      rc = CheckBias(fn, "d_dbias", a, grads->d_dbias, true, &regions);
    const struct {
      const char *name;
      const mfh_heads *v;
      int heads, tokens;
      bool written;
      mfh::HeadsView *to;
    } arrays[] = {{"out", &grads->out, a->heads, a->q_len, false, &t.out},
                  {"dout", &grads->dout, a->heads, a->q_len, false, &t.dout},
                  {"dq", &grads->dq, a->heads, a->q_len, true, &t.dq},
                  {"dk", &grads->dk, a->kv_heads, a->k_len, true, &t.dk},
                  {"dv", &grads->dv, a->kv_heads, a->k_len, true, &t.dv}};
    for (const auto &x : arrays)
      if (rc == MFH_OK && (x.v->p || !x.written))
        rc = CheckHeads(fn, x.name, a, *x.v, x.heads, x.tokens, x.written, &regions, x.to);
    if (rc != MFH_OK)
      return rc;
    const bool rows = a->batch > 0 && a->q_len > 0;
    if (rows && !grads->d_lse)
      return Invalid(fn, "null lse");
    if (!Aligned(grads->d_lse, 4))
      return Invalid(fn, "pointers must be aligned to their elements");
    const uint64_t need = mfh::AttentionBackwardWorkspace(t);
    rc = NeedWorkspace(fn, grads->d_workspace, grads->workspace_bytes, need);
    if (rc != MFH_OK)
      return rc;
    t.dbias = a->k_len > 0 ? grads->d_dbias : nullptr;
    if (!t.dq.p && !t.dk.p && !t.dv.p && !(rows && t.dbias))
      return MFH_OK;
    void *workspace = need > 0 ? grads->d_workspace : nullptr;
    AddFlat("d_lse", grads->d_lse, 4 * std::int64_t(a->batch) * a->heads * a->q_len, false,
            &regions);
    AddFlat("d_workspace", workspace, static_cast<std::int64_t>(need), true, &regions);
    rc = CheckApart(fn, regions);
    if (rc != MFH_OK)
      return rc;
    OnDevice on;
    const bool keys = a->k_len > 0;
    const Named ptrs[] = {{"q", t.q.p},
                          {"k", t.k.p},
                          {"v", t.v.p},
                          {"out", t.out.p},
                          {"dout", t.dout.p},
                          {"d_bias", keys && rows ? a->d_bias : nullptr},
                          {"d_q_lengths", a->d_q_lengths},
                          {"d_k_lengths", a->d_k_lengths},
                          {"d_lse", rows ? grads->d_lse : nullptr},
                          {"dq", t.dq.p},
                          {"dk", t.dk.p},
                          {"dv", t.dv.p},
                          {"d_dbias", rows ? t.dbias : nullptr},
                          {"d_workspace", workspace}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    rc = Enter(fn, a->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    t.bias_dtype = a->bias_dtype;
    t.bias_batch = a->bias_batch;
    t.bias_head = a->bias_head;
    t.bias_query = a->bias_query;
    t.lse = const_cast<float *>(grads->d_lse);
    t.workspace = workspace;
    std::string err;
    const hipError_t e = mfh::LaunchAttentionBackward(t, st, &err);
    return Done(fn, e, err);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

int mfh_adamw_set_create(const mfh_adamw_tensor *tensors, int n_tensors, int state_bits, int device,
                         mfh_adamw_set **out) {
  const char *fn = "mfh_adamw_set_create";
  if (!out || n_tensors < 0 || (n_tensors > 0 && !tensors) || device < -1)
    return Invalid(fn, "bad arguments");
  *out = nullptr;
  if (state_bits != 8 && state_bits != 32)
    return Invalid(fn, "state_bits must be 8 or 32");
  try {
    const bool eight = state_bits == 8;
    struct Range {
      std::uintptr_t begin, end;
      bool written;
    };
    std::vector<Range> ranges;
    std::int64_t total = 0;
    for (int i = 0; i < n_tensors; ++i) {
      const mfh_adamw_tensor &t = tensors[i];
      if (!KnownType(t.param_dtype) || !KnownType(t.grad_dtype) ||
          (t.copy && !KnownType(t.copy_dtype)))
        return Invalid(fn, "unknown dtype");
      if (!(t.lr_scale >= 0.f) || !Finite(t.lr_scale) || !(t.weight_decay >= 0.f) ||
          !Finite(t.weight_decay))
        return Invalid(fn, "lr_scale and weight_decay must be finite and >= 0");
      if (t.count == 0)
        continue;
      if (t.count > kMostElements || !t.param || !t.grad || !t.m || !t.v)
        return Invalid(fn, "a tensor without memory, or too large");
      if (eight != (t.m_scale != nullptr) || eight != (t.v_scale != nullptr))
        return Invalid(fn, "m_scale and v_scale go with states in 8 bits");
      const std::uintptr_t n = t.count, blocks = (n + mfh::kAdamBlock - 1) / mfh::kAdamBlock;
      const int state = eight ? 1 : 4;
      const struct {
        const void *p;
        std::uintptr_t n;
        int es;
        bool written;
      } arrays[] = {{t.param, n, mfh::DTypeBytes(t.param_dtype), true},
                    {t.grad, n, mfh::DTypeBytes(t.grad_dtype), false},
                    {t.m, n, state, true},
                    {t.v, n, state, true},
                    {t.m_scale, blocks, 4, true},
                    {t.v_scale, blocks, 4, true},
                    {t.copy, n, t.copy ? mfh::DTypeBytes(t.copy_dtype) : 1, true}};
      for (const auto &x : arrays) {
        if (!x.p)
          continue;
        if (!Aligned(x.p, x.es))
          return Invalid(fn, "pointers must be aligned to their elements");
        const std::uintptr_t b = mfh::Address(x.p);
        ranges.push_back({b, b + x.n * x.es, x.written});
        total += static_cast<std::int64_t>(x.n) * x.es;
      }
    }
    // In order of their beginning, a range meets an earlier one exactly when it
    // begins before the furthest end so far, of those written or (if it is
    // written itself) of any.
    std::sort(ranges.begin(), ranges.end(),
              [](const Range &a, const Range &b) { return a.begin < b.begin; });
    std::uintptr_t end_any = 0, end_written = 0;
    for (const Range &r : ranges) {
      if (r.begin < end_written || (r.written && r.begin < end_any))
        return Invalid(fn, "two arrays overlap, one of which is written");
      end_any = std::max(end_any, r.end);
      if (r.written)
        end_written = std::max(end_written, r.end);
    }

    int rc = NeedDevice(fn, device);
    if (rc != MFH_OK)
      return rc;
    int dev = device;
    for (int i = 0; i < n_tensors; ++i) {
      const mfh_adamw_tensor &t = tensors[i];
      if (t.count == 0)
        continue;
      const Named ptrs[] = {{"param", t.param},     {"grad", t.grad},       {"m", t.m}, {"v", t.v},
                            {"m_scale", t.m_scale}, {"v_scale", t.v_scale}, {"copy", t.copy}};
      for (const Named &p : ptrs) {
        rc = p.p ? PointerDevice(fn, p.name, p.p, dev, &dev) : MFH_OK;
        if (rc != MFH_OK)
          return rc;
      }
    }
    if (dev < 0) {
      const hipError_t e = hipGetDevice(&dev);
      if (e != hipSuccess)
        return HipError(fn, "hipGetDevice", e);
    }
    if (!IsGfx950(dev))
      return mfh::SetError(MFH_ERR_NO_DEVICE,
                           std::string(fn) + ": the device is not gfx950 (MI355X)");
    OnDevice on;
    hipError_t e = on.Set(dev);
    if (e != hipSuccess)
      return HipError(fn, "hipSetDevice", e);
    std::vector<mfh::AdamChunk> chunks;
    std::int64_t block = 0;
    for (int i = 0; i < n_tensors; ++i) {
      const mfh_adamw_tensor &t = tensors[i];
      const auto at_of = [](const void *p, uint64_t at, int es) -> void * {
        return p ? const_cast<char *>(static_cast<const char *>(p)) + at * es : nullptr;
      };
      for (uint64_t at = 0; at < t.count; at += mfh::kAdamChunk) {
        mfh::AdamChunk c{};
        c.param = at_of(t.param, at, mfh::DTypeBytes(t.param_dtype));
        c.grad = at_of(t.grad, at, mfh::DTypeBytes(t.grad_dtype));
        c.m = at_of(t.m, at, eight ? 1 : 4);
        c.v = at_of(t.v, at, eight ? 1 : 4);
        c.copy = at_of(t.copy, at, mfh::DTypeBytes(t.copy_dtype));
        c.m_scale = static_cast<float *>(at_of(t.m_scale, at / mfh::kAdamBlock, 4));
        c.v_scale = static_cast<float *>(at_of(t.v_scale, at / mfh::kAdamBlock, 4));
        c.first_block = block + static_cast<std::int64_t>(at / mfh::kAdamBlock);
        c.count = static_cast<std::int32_t>(std::min<uint64_t>(mfh::kAdamChunk, t.count - at));
        c.param_dtype = static_cast<std::uint8_t>(t.param_dtype);
        c.grad_dtype = static_cast<std::uint8_t>(t.grad_dtype);
        c.copy_dtype = static_cast<std::uint8_t>(t.copy_dtype);
        c.lr_scale = t.lr_scale;
        c.weight_decay = t.weight_decay;
        chunks.push_back(c);
      }
      block += static_cast<std::int64_t>((t.count + mfh::kAdamBlock - 1) / mfh::kAdamBlock);
    }
    auto set = std::make_unique<mfh_adamw_set>();
    set->device = dev;
    set->eight = eight;
    set->past = total > mfh::kAdamCachedBytes;
    set->n_chunks = static_cast<std::int64_t>(chunks.size());
    std::vector<mfh::ByteRange> memory;
    for (const Range &r : ranges)
      memory.push_back({r.begin, r.end});
    set->memory = mfh::Joined(std::move(memory));
    if (!chunks.empty()) {
      const size_t bytes = chunks.size() * sizeof(mfh::AdamChunk);
      e = hipMalloc(reinterpret_cast<void **>(&set->chunks), bytes);
      if (e != hipSuccess) {
        (void)hipGetLastError();
        return mfh::SetError(MFH_ERR_OUT_OF_MEMORY,
                             std::string(fn) + ": chunk list allocation failed");
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
    return mfh::SetError(MFH_ERR_OUT_OF_MEMORY, std::string(fn) + ": out of host memory");
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

void mfh_adamw_set_destroy(mfh_adamw_set *set) {
  if (!set)
    return;
  OnDevice on;
  (void)on.Set(set->device);
  if (set->chunks)
    (void)hipFree(set->chunks);
  delete set;
}

int mfh_adamw_step_device(const mfh_adamw_set *set, const mfh_adamw_step *step, void *stream) {
  const char *fn = "mfh_adamw_step_device";
  if (!set || !step)
    return Invalid(fn, "null argument");
  const auto beta = [](double b) { return b >= 0.0 && b < 1.0; };
  if (!(step->lr >= 0.0) || !std::isfinite(step->lr) || !beta(step->beta1) || !beta(step->beta2) ||
      !(step->eps >= 0.0) || !std::isfinite(step->eps))
    return Invalid(fn, "lr and eps must be finite and >= 0, beta1 and beta2 in [0, 1)");
  if (!(step->grad_scale > 0.0) || step->grad_scale > FLT_MAX || step->lr > FLT_MAX)
    return Invalid(fn, "grad_scale must be positive, and it and lr finite in 32 bits");
  if (step->step < 1)
    return Invalid(fn, "step must be >= 1");
  if ((step->skip_nonfinite != 0 && step->skip_nonfinite != 1) ||
      (step->stochastic != 0 && step->stochastic != 1))
    return Invalid(fn, "skip_nonfinite and stochastic must be 0 or 1");
  if (step->skip_nonfinite && !step->d_sumsq)
    return Invalid(fn, "skip_nonfinite needs d_sumsq");
  if (step->d_sumsq && !(step->max_norm >= 0.f))
    return Invalid(fn, "max_norm must be >= 0");
  if (!Aligned(step->d_sumsq, 8) || !Aligned(step->d_step, 8) || !Aligned(step->d_lr, 4))
    return Invalid(fn, "pointers must be aligned to their elements");
  if ((step->d_sumsq && mfh::Meets(set->memory, step->d_sumsq, 8)) ||
      (step->d_step && mfh::Meets(set->memory, step->d_step, 8)) ||
      (step->d_lr && mfh::Meets(set->memory, step->d_lr, 4)))
    return Invalid(fn, "d_sumsq, d_step or d_lr lies in a tensor");
  try {
    OnDevice on;
    const Named ptrs[] = {
        {"d_sumsq", step->d_sumsq}, {"d_step", step->d_step}, {"d_lr", step->d_lr}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = Enter(fn, set->device, ptrs, st, &on);
    if (rc != MFH_OK)
      return rc;
    mfh::AdamParams p;
    p.lr = step->lr;
    p.beta1 = step->beta1;
    p.beta2 = step->beta2;
    p.eps = step->eps;
    p.grad_scale = step->grad_scale;
    p.step = step->step;
    p.d_lr = step->d_lr;
    p.d_step = step->d_step;
    p.sumsq = step->d_sumsq;
    p.max_norm = step->max_norm;
    p.skip_nonfinite = step->skip_nonfinite != 0;
    p.stochastic = step->stochastic != 0;
    p.seed = step->seed;
    std::string err;
    const hipError_t e =
        mfh::LaunchAdamW(set->chunks, set->n_chunks, set->eight, set->past, p, st, &err);
    return Done(fn, e, err);
  } catch (const std::exception &e) {
    return Invalid(fn, e.what());
  }
}

}  // extern "C"
