// The C entry points of the learning operators (include/kgx.h): their checks of arguments, and the launch with the caller's
// current device restored.
#include "kgx_learn.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
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

// Vectors of floats, NULL where a call has none.
struct Floats {
  const char* name;
  const float* p;
};
void check_floats(std::initializer_list<Floats> vectors, const char* op) {
  for (const Floats& v : vectors)
    if (!aligned(v.p, 4)) bad(op, std::string(v.name) + " is not aligned to its elements");
}

// What a call reads or writes: `rows` rows of `width` bytes, `step` bytes apart (width <= step where there are several).
typedef __int128 wide;
struct Region {
  const char* name;
  wide begin, end;  // end: past its last byte; begin where there is nothing
  long long rows;
  wide width, step;
};
Region matrix(const char* name, const void* p, long long rows, long long width, long long ld, int size) {
  const wide begin = (wide)(uintptr_t)p, bytes = (wide)width * size, step = rows > 1 ? (wide)ld * size : bytes;
  return {name, begin, p && rows > 0 ? begin + (rows - 1) * step + bytes : begin, rows, bytes, step};
}
Region vector(const char* name, const void* p, long long n, int size = 4) { return matrix(name, p, 1, n, 0, size); }

// The least x >= 0 for which a x mod m is in [lo, hi], 0 < lo <= hi < m and 0 <= a < m; -1 where there is none. A multiple of a reaches lo before
// it passes m, or none does without passing m: a x in [lo + m y, hi + m y] then, and the least y is such a question of m y mod a.
wide first_within(wide a, wide m, wide lo, wide hi) {
  if (a == 0) return -1;
  const wide x = (lo + a - 1) / a;
  if (x * a <= hi) return x;
  // (No multiple of a is in [lo, hi]: -hi mod a is below -lo mod a, and neither is 0.)
  const wide y = first_within(m % a, a, (a - hi % a) % a, (a - lo % a) % a);
  return y < 0 ? -1 : (lo + m * y + a - 1) / a;
}

// Whether two regions share a byte: views side by side of one buffer do not, whatever their strides.
bool share(const Region& a, const Region& b) {
  if (b.begin >= a.end || a.begin >= b.end || a.begin == a.end || b.begin == b.end) return false;
  const wide at = b.begin - a.begin;
  // b's rows first ... last touch a's extent.
  const wide first = at + b.width > 0 ? 0 : (-at - b.width) / b.step + 1, last = std::min((wide)b.rows - 1, (a.end - 1 - b.begin) / b.step);
  if (first > last) return false;
  // One that begins within a's extent lies between two of a's rows if its start is in [a.width, a.step - b.width] of one's.
  const wide start = at + first * b.step;
  if (start < 0 || a.width > a.step - b.width) return true;
  const wide room = a.width + b.width - 2, r = (start + b.width - 1) % a.step;
  if (r <= room) return true;
  const wide next = first_within(b.step % a.step, a.step, a.step - r, a.step - r + room);
  return next >= 0 && next <= last - first;
}

// Outputs, and what a call has of its own until it has run, share no memory with anything else of the call.
void check_apart(std::initializer_list<Region> out, std::initializer_list<Region> in, const char* op) {
  for (const Region* o = out.begin(); o != out.end(); o++) {
    for (const Region* r = o + 1; r != out.end(); r++)
      if (share(*o, *r)) bad(op, std::string(o->name) + " must not overlap " + r->name);
    for (const Region& r : in)
      if (share(*o, r)) bad(op, std::string(o->name) + " must not overlap " + r.name);
  }
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

void check_distill(const kg_distill_loss_args& a) {
  const char* op = "distillation loss";
  need(a.rows >= 0 && a.rows <= kMaxRows && a.columns >= 1 && a.columns <= kMaxColumns, op, "rows must be in [0, 2^30] and columns in [1, 2^30]");
  need(a.k >= 1 && a.k <= KG_DISTILL_MAX_K, op, "k must be in [1, 1024]");
  check_type(a.type, op);
  check_type(a.top_type, op);
  need(a.logit_scale >= 0x1p-64 && a.logit_scale <= 0x1p64, op, "logit_scale must be positive, in [2^-64, 2^64]");
  if (!a.rows) return;
  check_rows(a.logits, a.rows, a.columns, a.ld, a.type, op, "logits");
  check_rows(a.top_index, a.rows, a.k, a.ld_index, KG_PRECISION_F32, op, "top_index");  // (4 bytes too)
  check_rows(a.top_logits, a.rows, a.k, a.ld_top, a.top_type, op, "top_logits");
  if (a.grad) check_rows(a.grad, a.rows, a.columns, a.ld_grad, a.type, op, "grad");
  if (a.legal) need(a.ld_legal >= (a.rows > 1 ? a.columns : 0), op, "the row stride of legal is less than its row");
  need(a.loss, op, "null argument");
  check_floats({{"loss", a.loss}, {"weight", a.weight}, {"teacher_lse", a.teacher_lse}}, op);
  const size_t work = kgx::distill_loss_workspace(a.rows, a.columns, a.k);
  if (work) {
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  }
  const int size = (int)size_of(a.type);
  check_apart({matrix("grad", a.grad, a.rows, a.columns, a.ld_grad, size), vector("loss", a.loss, a.rows), vector("workspace", a.workspace, work, 1)},
              {matrix("logits", a.logits, a.rows, a.columns, a.ld, size), matrix("legal", a.legal, a.rows, a.columns, a.ld_legal, 1),
               matrix("top_index", a.top_index, a.rows, a.k, a.ld_index, 4),
               matrix("top_logits", a.top_logits, a.rows, a.k, a.ld_top, (int)size_of(a.top_type)), vector("teacher_lse", a.teacher_lse, a.rows),
               vector("weight", a.weight, a.rows)},
              op);
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

void check_layer_norm(const kg_layer_norm_args& a, bool backward) {
  const char* op = backward ? "layer norm backward" : "layer norm";
  need(a.rows >= 0 && a.rows <= kMaxRows && a.channels >= 1 && a.channels <= kMaxColumns, op,
       "rows must be in [0, 2^30] and channels in [1, 2^30]");
  check_type(a.type, op);
  if (!backward) need(usable_eps(a.eps), op, "eps must be positive, at least 2^-126");
  const Region dgamma = vector("dgamma", a.dgamma, a.channels), dbeta = vector("dbeta", a.dbeta, a.channels);
  if (backward) {  // (written for no rows too: 0)
    check_floats({{"dgamma", a.dgamma}, {"dbeta", a.dbeta}}, op);
    check_apart({dgamma, dbeta}, {}, op);
  }
  if (!a.rows) return;
  need((a.mean || a.rms) && a.rstd, op, "mean or rstd is null");
  check_floats({{"gamma", a.gamma}, {"mean", a.rms ? nullptr : a.mean}, {"rstd", a.rstd}}, op);
  if (!backward) check_floats({{"beta", a.beta}}, op);
  check_rows(a.x, a.rows, a.channels, a.ldx, a.type, op, "x");
  if (backward) {
    check_rows(a.dy, a.rows, a.channels, a.lddy, a.type, op, "dy");
    check_rows(a.dx, a.rows, a.channels, a.lddx, a.type, op, "dx");
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  } else {
    check_rows(a.y, a.rows, a.channels, a.ldy, a.type, op, "y");
  }
  const int size = (int)size_of(a.type);
  const Region x = matrix("x", a.x, a.rows, a.channels, a.ldx, size), gamma = vector("gamma", a.gamma, a.channels);
  const Region mean = vector("mean", a.rms ? nullptr : a.mean, a.rows), rstd = vector("rstd", a.rstd, a.rows);
  if (backward)
    check_apart({matrix("dx", a.dx, a.rows, a.channels, a.lddx, size), dgamma, dbeta,
                 vector("workspace", a.workspace, kgx::layer_norm_workspace(a.rows, a.channels), 1)},
                {x, matrix("dy", a.dy, a.rows, a.channels, a.lddy, size), gamma, mean, rstd}, op);
  else
    check_apart({matrix("y", a.y, a.rows, a.channels, a.ldy, size), mean, rstd}, {x, gamma, vector("beta", a.beta, a.channels)}, op);
}

void check_embedding(const kg_embedding_args& a, bool backward) {
  const char* op = backward ? "embedding backward" : "embedding";
  need(a.count >= 0 && a.count <= kMaxRows && a.vocab >= 1 && a.vocab <= kMaxRows && a.channels >= 1 && a.channels <= kMaxColumns, op,
       "count must be in [0, 2^30], vocab and channels in [1, 2^30]");
  check_type(a.type, op);
  need(finite_float(a.scale), op, "scale must be finite in float");
  if (backward) {
    need(a.grad_type == a.type || a.grad_type == KG_PRECISION_F32, op, "grad_type must be the type of dy or float");
    if (a.count || !a.accumulate) check_rows(a.grad, a.vocab, a.channels, a.ld_grad, a.grad_type, op, "grad");
  }
  if (!a.count) return;
  need(a.tokens && aligned(a.tokens, 4), op, "tokens is null or not aligned to its elements");
  if (backward) {
    check_rows(a.dy, a.count, a.channels, a.ld_dy, a.type, op, "dy");
    need(a.workspace, op, "workspace is null");
    need(aligned(a.workspace, 16), op, "workspace is not aligned to 16 bytes");
  } else {
    check_rows(a.table, a.vocab, a.channels, a.ld_table, a.type, op, "table");
    check_rows(a.y, a.count, a.channels, a.ld_y, a.type, op, "y");
  }
  const int size = (int)size_of(a.type);
  const Region tokens = vector("tokens", a.tokens, a.count);
  if (backward)
    check_apart({matrix("grad", a.grad, a.vocab, a.channels, a.ld_grad, (int)size_of(a.grad_type)),
                 vector("workspace", a.workspace, kgx::embedding_backward_workspace(a.count, a.vocab, a.channels), 1)},
                {matrix("dy", a.dy, a.count, a.channels, a.ld_dy, size), tokens}, op);
  else
    check_apart({matrix("y", a.y, a.count, a.channels, a.ld_y, size)}, {matrix("table", a.table, a.vocab, a.channels, a.ld_table, size), tokens}, op);
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

// (Sizes that no call takes need none, and would overflow the sums.)
size_t kg_distill_loss_workspace(int rows, int columns, int k) {
  if (rows < 1 || rows > kMaxRows || columns < 1 || columns > kMaxColumns || k < 1 || k > KG_DISTILL_MAX_K) return 0;
  return kgx::distill_loss_workspace(rows, columns, k);
}

int kg_distill_loss(int device, void* stream, const kg_distill_loss_args* args) {
  return guarded([&] {
    need(args, "distillation loss", "null argument");
    check_distill(*args);
    if (!args->rows) return;
    OnDevice on(device, "distillation loss");
    kgx::launch_distill_loss(*args, (hipStream_t)stream);
  });
}

size_t kg_layer_norm_workspace(int rows, int channels) {
  if (rows < 1 || rows > kMaxRows || channels < 1 || channels > kMaxColumns) return 0;
  return kgx::layer_norm_workspace(rows, channels);
}

int kg_layer_norm(int device, void* stream, const kg_layer_norm_args* args) {
  return guarded([&] {
    need(args, "layer norm", "null argument");
    check_layer_norm(*args, false);
    if (!args->rows) return;
    OnDevice on(device, "layer norm");
    kgx::launch_layer_norm(*args, (hipStream_t)stream);
  });
}

int kg_layer_norm_backward(int device, void* stream, const kg_layer_norm_args* args) {
  return guarded([&] {
    need(args, "layer norm backward", "null argument");
    check_layer_norm(*args, true);
    OnDevice on(device, "layer norm backward");
    kgx::launch_layer_norm_backward(*args, (hipStream_t)stream);
  });
}

size_t kg_embedding_backward_workspace(int count, int vocab, int channels) {
  if (count < 1 || count > kMaxRows || vocab < 1 || vocab > kMaxRows || channels < 1 || channels > kMaxColumns) return 0;
  return kgx::embedding_backward_workspace(count, vocab, channels);
}

int kg_embedding(int device, void* stream, const kg_embedding_args* args) {
  return guarded([&] {
    need(args, "embedding", "null argument");
    check_embedding(*args, false);
    if (!args->count) return;
    OnDevice on(device, "embedding");
    kgx::launch_embedding(*args, (hipStream_t)stream);
  });
}

int kg_embedding_backward(int device, void* stream, const kg_embedding_args* args) {
  return guarded([&] {
    need(args, "embedding backward", "null argument");
    check_embedding(*args, true);
    if (!args->count && args->accumulate) return;
    OnDevice on(device, "embedding backward");
    kgx::launch_embedding_backward(*args, (hipStream_t)stream);
  });
}

}  // extern "C"
