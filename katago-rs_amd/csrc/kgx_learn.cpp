// The C entry points of the learning operators (include/kgx.h): their checks of arguments, and the launch with the caller's
// current device restored.
#include "kgx_learn.h"

#include <cmath>
#include <cstdint>
#include <limits>
#include <string>

#include "kgx_error.h"
#include "kgx_kernels.h"

namespace {

using kgx::guarded;

[[noreturn]] void bad(const char* op, const std::string& what) { throw std::runtime_error(std::string("kgx ") + op + ": " + what); }
void need(bool ok, const char* op, const char* what) {
  if (!ok) bad(op, what);
}

void hip(hipError_t e, const char* op) {
  if (e != hipSuccess) bad(op, hipGetErrorString(e));
}

// `device` current for a scope.
class OnDevice {
 public:
  OnDevice(int device, const char* op) {
    hip(hipGetDevice(&before_), op);
    if (device != before_) {
      hip(hipSetDevice(device), op);
      changed_ = true;
    }
  }
  ~OnDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

void check_type(int type, const char* op) {
  need(type == KG_PRECISION_F32 || type == KG_PRECISION_F16 || type == KG_PRECISION_BF16, op, "unknown element type");
}
bool aligned(const void* p, size_t to) { return ((uintptr_t)p) % to == 0; }
size_t size_of(int type) { return type == KG_PRECISION_F32 ? 4 : 2; }
bool finite_at_least(double v, double least) { return std::isfinite(v) && v >= least; }
bool finite_float(double v) { return std::isfinite((float)v); }
// An eps whose reciprocal, and the square of whose root's, are finite floats.
bool usable_eps(double v) { return v >= (double)std::numeric_limits<float>::min() && finite_float(v); }

// A matrix of `rows` rows of `width` elements, `ld` apart.
void check_rows(const void* p, long long rows, long long width, long long ld, int type, const char* op, const char* name) {
  if (!p) bad(op, std::string(name) + " is null");
  if (rows > 1 && ld < width) bad(op, std::string("the row stride of ") + name + " is less than its row");
  if (ld < 0 || (rows > 1 && ld > std::numeric_limits<long long>::max() / 8 / rows)) bad(op, std::string("the row stride of ") + name + " is out of range");
  if (!aligned(p, size_of(type))) bad(op, std::string(name) + " is not aligned to its elements");
}

constexpr int kMaxRows = 1 << 30;     // a workgroup's step over them stays below 2^31
constexpr int kMaxColumns = 1 << 30;  // a row's element indices have 31 bits, past its end too

void check_policy(const kg_policy_loss_args& a) {
  const char* op = "policy loss";
  need(a.rows >= 0 && a.rows <= kMaxRows && a.columns >= 1 && a.columns <= kMaxColumns, op, "rows must be in [0, 2^30] and columns in [1, 2^30]");
  check_type(a.type, op);
  need(a.logit_scale >= 0x1p-64 && a.logit_scale <= 0x1p64, op, "logit_scale must be positive, in [2^-64, 2^64]");
  need(finite_at_least(a.clip_low, 0) && a.clip_low < 1 && finite_at_least(a.clip_high, 0), op,
       "clip_low must be in [0, 1) and clip_high at least 0");
  need(finite_float(a.kl_coef), op, "kl_coef must be finite in float");
  need(!(a.ref_logits && a.ref_logp), op, "give ref_logits or ref_logp, not both");
  if (!a.rows) return;
  check_rows(a.logits, a.rows, a.columns, a.ld, a.type, op, "logits");
  if (a.ref_logits) check_rows(a.ref_logits, a.rows, a.columns, a.ld_ref, a.type, op, "ref_logits");
  if (a.grad) check_rows(a.grad, a.rows, a.columns, a.ld_grad, a.type, op, "grad");
  if (a.legal) need(a.ld_legal >= (a.rows > 1 ? a.columns : 0), op, "the row stride of legal is less than its row");
  need(a.action && a.old_logp && a.advantage && a.loss && a.logp && a.kl, op, "null argument");
  need(a.grad != a.logits && (!a.grad || a.grad != a.ref_logits), op, "grad must not overlap an input");
  if (kgx::policy_loss_workspace(a.rows, a.columns)) {
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  }
}

void check_preference(const kg_preference_loss_args& a) {
  const char* op = "preference loss";
  need(a.rows >= 0 && a.rows <= kMaxRows && a.columns >= 1 && a.columns <= kMaxColumns && a.pairs >= 0, op,
       "rows must be in [0, 2^30], columns in [1, 2^30] and pairs at least 0");
  need(a.pairs <= std::numeric_limits<int>::max() / 2 - 1, op, "too many pairs");
  check_type(a.type, op);
  need(std::isfinite(a.beta) && a.beta > 0, op, "beta must be positive");
  need(finite_at_least(a.label_smoothing, 0) && a.label_smoothing <= 0.5, op, "label_smoothing must be in [0, 0.5]");
  need(a.offsets, op, "offsets is null");
  if (a.rows) {
    check_rows(a.logits, a.rows, a.columns, a.ld, a.type, op, "logits");
    if (a.grad) check_rows(a.grad, a.rows, a.columns, a.ld_grad, a.type, op, "grad");
    need(a.grad != a.logits, op, "grad must not overlap an input");
    need(a.label, op, "label is null");
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  }
  if (a.pairs) need(a.ref_logp && a.loss && a.margin && a.seq_logp, op, "null argument");
}

void check_state(const kg_adamw_state& s, const char* op) {
  need(s.state_bits == 8 || s.state_bits == 32, op, "state_bits must be 8 or 32");
  need(s.m && s.v, op, "the moments are null");
  if (s.state_bits == 8) need(s.m_exp && s.v_exp, op, "the blocks' exponents are null");
  else need(aligned(s.m, 4) && aligned(s.v, 4), op, "the moments are not aligned to their elements");
}

double step_size(const kg_adamw_hyper& h) { return h.lr / (1.0 - std::pow(h.beta1, (double)h.step)); }

void check_hyper(const kg_adamw_hyper& h) {
  const char* op = "AdamW";
  need(finite_float(h.lr), op, "lr must be finite in float");
  need(h.beta1 >= 0 && h.beta1 < 1 && h.beta2 >= 0 && h.beta2 < 1, op, "beta1 and beta2 must be in [0, 1)");
  need(usable_eps(h.eps), op, "eps must be positive, at least 2^-126");
  need(finite_float(h.grad_scale), op, "grad_scale must be finite in float");
  need(h.step >= 1, op, "step counts from 1");
  need(finite_float(step_size(h)), op, "lr / (1 - beta1^step) must be finite in float");
}

kg_adamw_values_t values_of(const kg_adamw_hyper& h) {
  kg_adamw_values_t v;
  const double t = (double)h.step;
  v.lr = (float)h.lr;
  v.beta1 = (float)h.beta1;
  v.beta1_rest = (float)(1.0 - h.beta1);
  v.beta2 = (float)h.beta2;
  v.beta2_rest = (float)(1.0 - h.beta2);
  v.eps = (float)h.eps;
  v.grad_scale = (float)h.grad_scale;
  v.step_size = (float)step_size(h);
  v.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(h.beta2, t)));
  v.seed = h.seed;
  return v;
}

constexpr int kMaxNormGroups = 2048;

void check_norm(const kg_group_norm_args& a, bool backward) {
  const char* op = backward ? "group norm backward" : "group norm";
  need(a.batch >= 0 && a.points >= 0, op, "batch and points must be at least 0");
  need(a.channels >= 1 && a.groups >= 1 && a.channels % a.groups == 0, op, "channels must be a multiple of groups");
  need(a.groups <= kMaxNormGroups, op, "at most 2048 groups are supported");
  need((long long)a.batch * a.points <= std::numeric_limits<int>::max() && (long long)a.batch * a.groups <= std::numeric_limits<int>::max(),
       op, "batch x points or batch x groups is out of range");
  check_type(a.type, op);
  need(a.act >= KG_ACT_IDENTITY && a.act <= KG_ACT_SILU, op, "unknown activation");
  const long long rows = (long long)a.batch * a.points;
  if (!backward) need(usable_eps(a.eps), op, "eps must be positive, at least 2^-126");
  if (a.batch) need(a.mean && a.rstd, op, "mean or rstd is null");
  if (rows) {
    check_rows(a.x, rows, a.channels, a.ldx, a.type, op, "x");
    if (backward) {
      check_rows(a.dy, rows, a.channels, a.lddy, a.type, op, "dy");
      check_rows(a.dx, rows, a.channels, a.lddx, a.type, op, "dx");
      need(a.dx != a.x && a.dx != a.dy, op, "dx must not overlap an input");
    } else {
      check_rows(a.y, rows, a.channels, a.ldy, a.type, op, "y");
      need(a.y != a.x, op, "y must not overlap x");
    }
  }
  if (a.batch) {
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  }
  need(kgx::group_norm_fits(a), op, "batch x groups is out of range");
}

}  // namespace

extern "C" {

int kg_policy_loss(int device, void* stream, const kg_policy_loss_args* args) {
  return guarded([&] {
    need(args, "policy loss", "null argument");
    check_policy(*args);
    if (!args->rows) return;
    OnDevice on(device, "policy loss");
    kgx::launch_policy_loss(*args, (hipStream_t)stream);
  });
}

size_t kg_policy_loss_workspace(int rows, int columns) { return kgx::policy_loss_workspace(rows, columns); }

size_t kg_preference_loss_workspace(int rows) { return kgx::preference_loss_workspace(rows); }

int kg_preference_loss(int device, void* stream, const kg_preference_loss_args* args) {
  return guarded([&] {
    need(args, "preference loss", "null argument");
    check_preference(*args);
    if (!args->rows && !args->pairs) return;
    OnDevice on(device, "preference loss");
    kgx::launch_preference_loss(*args, (hipStream_t)stream);
  });
}

int kg_adamw_values(const kg_adamw_hyper* hyper, kg_adamw_values_t* out) {
  return guarded([&] {
    need(hyper && out, "AdamW", "null argument");
    check_hyper(*hyper);
    *out = values_of(*hyper);
  });
}

int kg_adamw_step(int device, void* stream, int count, const kg_adamw_tensor* tensors, const kg_adamw_state* state,
                  const kg_adamw_hyper* hyper, const kg_adamw_values_t* values) {
  return guarded([&] {
    const char* op = "AdamW";
    need(count >= 0, op, "count must be at least 0");
    need((tensors || !count) && state && hyper, op, "null argument");
    check_hyper(*hyper);
    need(aligned(values, 4), op, "values is not aligned to its floats");
    if (!count) return;
    check_state(*state, op);
    for (int i = 0; i < count; i++) {
      const kg_adamw_tensor& t = tensors[i];
      const auto at = [i] { return "tensor " + std::to_string(i) + ": "; };
      check_type(t.param_type, op);
      check_type(t.grad_type, op);
      if (t.elements < 0 || t.first_block < 0 || t.elements > (1ll << 46) || t.first_block > (1ll << 38)) bad(op, at() + "size out of range");
      if (!finite_float(t.weight_decay)) bad(op, at() + "weight_decay must be finite in float");
      if (!t.elements) continue;
      if (!t.param || !t.grad) bad(op, at() + "null argument");
      if (!aligned(t.param, size_of(t.param_type)) || !aligned(t.grad, size_of(t.grad_type)) || !aligned(t.master, 4))
        bad(op, at() + "not aligned to its elements");
    }
    OnDevice on(device, op);
    kgx::launch_adamw(count, tensors, *state, values_of(*hyper), values, (hipStream_t)stream);
  });
}

int kg_adamw_moments(int device, void* stream, long long blocks, const kg_adamw_state* state, int type, void* m, void* root) {
  return guarded([&] {
    const char* op = "AdamW";
    need(state && blocks >= 0, op, "null argument");
    check_type(type, op);
    if (!blocks) return;
    check_state(*state, op);
    need(m && root, op, "null argument");
    need(aligned(m, size_of(type)) && aligned(root, size_of(type)), op, "not aligned to its elements");
    OnDevice on(device, op);
    kgx::launch_adamw_moments(blocks, *state, type, m, root, (hipStream_t)stream);
  });
}

size_t kg_group_norm_workspace(int batch, int points, int channels, int groups, int backward) {
  if (batch < 0 || points < 0 || channels < 1 || groups < 1 || groups > kMaxNormGroups) return 0;  // (no call takes those)
  return kgx::group_norm_workspace(batch, points, channels, groups, backward != 0);
}

int kg_group_norm(int device, void* stream, const kg_group_norm_args* args) {
  return guarded([&] {
    need(args, "group norm", "null argument");
    check_norm(*args, false);
    if (!args->batch) return;
    OnDevice on(device, "group norm");
    kgx::launch_group_norm(*args, (hipStream_t)stream);
  });
}

int kg_group_norm_backward(int device, void* stream, const kg_group_norm_args* args) {
  return guarded([&] {
    need(args, "group norm backward", "null argument");
    check_norm(*args, true);
    OnDevice on(device, "group norm backward");
    kgx::launch_group_norm_backward(*args, (hipStream_t)stream);
  });
}

}  // extern "C"
