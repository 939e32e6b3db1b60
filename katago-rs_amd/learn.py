"""Learning from the network's answers: the operators of include/kgx.h's last section on torch tensors of a GPU.

- `policy_loss`: the clipped policy loss with a KL term on rows of logits (a network's policy rows with their legal moves,
  or tokens), and its gradient;
- `preference_loss`: pairs of lines of moves or token sequences, the better against the worse, and its gradient;
- `AdamW`: one step over many tensors at once, moments in 32 or in 8 bits;
- `group_norm` and `group_norm_backward`: group norm with an activation on channels-last rows under the board mask.

The calls run on torch's current stream of the tensors' device and do not wait. They take part in no autograd graph: gradients
are returned. There is no other compute path, and a call that the library refuses raises KgError; a tensor of another shape,
type or device than the call needs raises ValueError. A network's own policy rows come from Handle.policy_rows:

    rows = torch.as_tensor(handle.policy_rows(n), device="cuda")   # [n, 362], inside the raw rows
    r = learn.policy_loss(rows, actions, old_logp, advantage, legal=legal, kl_coef=0.1, ref_logits=before)

torch has to be imported before the library is loaded (importing this module first does that): both use the process's one HIP
runtime.
"""

import collections
import ctypes

import numpy as np
import torch

from . import KgError, PRECISION_BF16, PRECISION_F16, PRECISION_F32, _check, lib

TYPES = {torch.float32: PRECISION_F32, torch.float16: PRECISION_F16, torch.bfloat16: PRECISION_BF16}
ACTS = {"identity": 0, "relu": 1, "mish": 2, "silu": 3}
BLOCK = 256  # KG_ADAMW_BLOCK

PolicyLoss = collections.namedtuple("PolicyLoss", ["loss", "logp", "kl", "grad"])
PreferenceLoss = collections.namedtuple("PreferenceLoss", ["loss", "margin", "seq_logp", "grad"])

_vp, _ci, _ll, _cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double


class _PolicyArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("columns", _ci), ("type", _ci), ("logits", _vp), ("ld", _ll), ("legal", _vp),
                ("ld_legal", _ll), ("action", _vp), ("old_logp", _vp), ("advantage", _vp), ("weight", _vp),
                ("ref_logits", _vp), ("ld_ref", _ll), ("ref_logp", _vp), ("logit_scale", _cd), ("clip_low", _cd),
                ("clip_high", _cd), ("kl_coef", _cd), ("loss", _vp), ("logp", _vp), ("kl", _vp), ("grad", _vp),
                ("ld_grad", _ll)]


class _PreferenceArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("columns", _ci), ("type", _ci), ("logits", _vp), ("ld", _ll), ("label", _vp),
                ("pairs", _ci), ("offsets", _vp), ("ref_logp", _vp), ("weight", _vp), ("beta", _cd),
                ("label_smoothing", _cd), ("average", _ci), ("loss", _vp), ("margin", _vp), ("seq_logp", _vp),
                ("grad", _vp), ("ld_grad", _ll), ("workspace", _vp)]


class _NormArgs(ctypes.Structure):
    _fields_ = [("batch", _ci), ("points", _ci), ("channels", _ci), ("groups", _ci), ("type", _ci), ("act", _ci),
                ("eps", _cd), ("x", _vp), ("ldx", _ll), ("mask", _vp), ("gamma", _vp), ("beta", _vp), ("mean", _vp),
                ("rstd", _vp), ("workspace", _vp), ("y", _vp), ("ldy", _ll), ("dy", _vp), ("lddy", _ll), ("dx", _vp),
                ("lddx", _ll), ("dgamma", _vp), ("dbeta", _vp)]


class _AdamTensor(ctypes.Structure):
    _fields_ = [("param", _vp), ("grad", _vp), ("master", _vp), ("elements", _ll), ("first_block", _ll),
                ("weight_decay", _cd), ("param_type", _ci), ("grad_type", _ci)]


class _AdamHyper(ctypes.Structure):
    _fields_ = [("lr", _cd), ("beta1", _cd), ("beta2", _cd), ("eps", _cd), ("grad_scale", _cd), ("step", _ll),
                ("seed", ctypes.c_uint)]


class _AdamState(ctypes.Structure):
    _fields_ = [("state_bits", _ci), ("m", _vp), ("v", _vp), ("m_exp", _vp), ("v_exp", _vp)]


class AdamValues(ctypes.Structure):
    """kg_adamw_values_t: the scalars of a step, as a captured step reads them from device memory."""
    _fields_ = [(f, ctypes.c_float) for f in ("lr", "beta1", "beta1_rest", "beta2", "beta2_rest", "eps", "grad_scale",
                                              "step_size", "root_scale")] + [("seed", ctypes.c_uint)]


_one_runtime = False


def _library():
    """The library, once it is certain that torch and it share one HIP runtime."""
    global _one_runtime
    L = lib()
    if not _one_runtime:
        with open("/proc/self/maps") as f:
            found = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(found) > 1:
            raise KgError("two HIP runtimes are loaded (%s): import torch before the library is loaded" %
                          ", ".join(sorted(found)))
        _one_runtime = True
    return L


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _rows(t, name, like=None):
    """(pointer, row stride) of a matrix on the GPU with unit column stride; `like`: of that shape, type and device."""
    if t.dim() != 2 or t.dtype not in TYPES or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be [rows, columns] of float32, float16 or bfloat16 with contiguous columns")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the shape, type and device of the logits")
    return t.data_ptr(), t.stride(0)


def _vector(t, n, dtype, name, device):
    """Pointer of a contiguous vector of n elements on `device`; None for None."""
    if t is None:
        return None
    if t.shape != (n,) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} {str(dtype)[6:]} on {device}")
    return t.data_ptr()


def policy_loss(logits, actions, old_logp, advantage, *, legal=None, weight=None, logit_scale=1.0, clip=(0.2, 0.2),
                kl_coef=0.0, ref_logits=None, ref_logp=None, want_grad=True, grad=None):
    """The clipped policy loss of each row with its KL term, and the gradient of their sum (kg_policy_loss).

    logits [n, v] (rows may be strided); actions [n] int32, outside [0, v) for padding; old_logp, advantage, weight [n]
    float32; legal [n, v] bool or uint8; clip (low, high): the ratio counts within [1 - low, 1 + high]; the KL term is the full
    one to ref_logits [n, v], or the estimate from ref_logp [n]. Returns loss, logp and kl [n] float32 and grad [n, v] of
    the logits' type (into `grad` when given; None without want_grad)."""
    ptr, ld = _rows(logits, "logits")
    n, v = logits.shape
    dev = logits.device
    lg, ld_lg = None, 0
    if legal is not None:
        if legal.shape != (n, v) or legal.dtype not in (torch.bool, torch.uint8) or legal.device != dev or \
                (legal.stride(1) != 1 and v > 1):
            raise ValueError(f"legal must be [{n}, {v}] bool or uint8 on {dev} with contiguous columns")
        lg, ld_lg = legal.data_ptr(), legal.stride(0)
    ref, ld_ref = (None, 0) if ref_logits is None else _rows(ref_logits, "ref_logits", logits)
    if grad is None and want_grad:
        grad = torch.empty(n, v, dtype=logits.dtype, device=dev)
    g, ld_g = (None, 0) if grad is None else _rows(grad, "grad", logits)
    out = torch.empty(3, n, dtype=torch.float32, device=dev)
    o = out.data_ptr()
    low, high = clip
    args = _PolicyArgs(n, v, TYPES[logits.dtype], ptr, ld, lg, ld_lg, _vector(actions, n, torch.int32, "actions", dev),
                       _vector(old_logp, n, torch.float32, "old_logp", dev),
                       _vector(advantage, n, torch.float32, "advantage", dev),
                       _vector(weight, n, torch.float32, "weight", dev), ref, ld_ref,
                       _vector(ref_logp, n, torch.float32, "ref_logp", dev), logit_scale, low, high, kl_coef, o, o + 4 * n,
                       o + 8 * n, g, ld_g)
    _check(_library().kg_policy_loss(dev.index, _stream(dev), ctypes.byref(args)))
    return PolicyLoss(out[0], out[1], out[2], grad)


def preference_loss(logits, labels, offsets, ref_logp, *, beta=0.1, label_smoothing=0.0, average=False, weight=None,
                    want_grad=True, grad=None):
    """The preference loss of pairs of sequences packed in rows of logits, and the gradient of its sum (kg_preference_loss).

    logits [t, v] (rows may be strided); labels [t] int32, outside [0, v) where a row is not counted; offsets [2 p + 1] int32:
    sequence q is rows [offsets[q], offsets[q + 1]), and pair i prefers sequence 2 i to 2 i + 1; ref_logp [2 p] float32: the
    sequences' log-probabilities (means with `average`) under the reference; weight [p] float32. Returns loss and margin [p],
    seq_logp [2 p] and grad [t, v] of the logits' type (into `grad` when given; None without want_grad)."""
    ptr, ld = _rows(logits, "logits")
    t, v = logits.shape
    dev = logits.device
    if offsets.dim() != 1 or offsets.shape[0] % 2 == 0:
        raise ValueError("offsets must be a vector of an odd length")
    p = offsets.shape[0] // 2
    if grad is None and want_grad:
        grad = torch.empty(t, v, dtype=logits.dtype, device=dev)
    g, ld_g = (None, 0) if grad is None else _rows(grad, "grad", logits)
    L = _library()
    out = torch.empty(4 * p, dtype=torch.float32, device=dev)
    work = torch.empty(L.kg_preference_loss_workspace(t), dtype=torch.uint8, device=dev)
    o = out.data_ptr()
    args = _PreferenceArgs(t, v, TYPES[logits.dtype], ptr, ld, _vector(labels, t, torch.int32, "labels", dev), p,
                           _vector(offsets, 2 * p + 1, torch.int32, "offsets", dev),
                           _vector(ref_logp, 2 * p, torch.float32, "ref_logp", dev),
                           _vector(weight, p, torch.float32, "weight", dev), beta, label_smoothing, bool(average), o, o + 4 * p,
                           o + 8 * p, g, ld_g, work.data_ptr())
    _check(L.kg_preference_loss(dev.index, _stream(dev), ctypes.byref(args)))
    return PreferenceLoss(out[:p], out[p:2 * p], out[2 * p:], grad)


def _points(t, name):
    """(pointer, row stride) of [batch, ..., channels] whose points lie evenly spaced."""
    if t.dim() < 2 or t.dtype not in TYPES:
        raise ValueError(f"{name} must be [batch, ..., channels] of float32, float16 or bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if not t.numel():
        return t.data_ptr(), t.shape[-1]
    ld = None
    span = 1
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size != 1:
            if ld is None:
                ld = stride
            elif stride != ld * span:
                raise ValueError(f"the points of {name} must be evenly spaced")
            span *= size
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous channels")
    return t.data_ptr(), t.shape[-1] if ld is None else ld


def _norm_shape(x, groups, gamma, beta, mask, act):
    if x.dim() < 2 or act not in ACTS:
        raise ValueError(f"x must be [batch, ..., channels] and act one of {', '.join(ACTS)}")
    batch, channels = x.shape[0], x.shape[-1]
    points = 1
    for s in x.shape[1:-1]:
        points *= s
    dev = x.device
    if mask is not None:
        if mask.shape != x.shape[:-1] or mask.dtype != torch.float32 or mask.device != dev or not mask.is_contiguous():
            raise ValueError(f"mask must be contiguous float32 of shape {tuple(x.shape[:-1])} on {dev}")
        mask = mask.data_ptr()
    return (batch, points, channels, int(groups), mask, _vector(gamma, channels, torch.float32, "gamma", dev),
            _vector(beta, channels, torch.float32, "beta", dev))


def group_norm(x, groups, gamma=None, beta=None, *, mask=None, eps=1e-5, act="identity", y=None):
    """act(group norm of x) on channels-last x [batch, ..., channels] over the points with a nonzero mask [batch, ...]
    (kg_group_norm). Returns y (into `y` when given; 0 where the mask is 0), and mean and rstd [batch, groups]."""
    ptr, ld = _points(x, "x")
    b, p, c, g, mk, gm, bt = _norm_shape(x, groups, gamma, beta, mask, act)
    if y is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
        raise ValueError("y must have the shape, type and device of x")
    yp, ldy = _points(y, "y")
    L = _library()
    stats = torch.empty(2, b, max(g, 0), dtype=torch.float32, device=x.device)
    work = torch.empty(L.kg_group_norm_workspace(b, p, c, g, 0), dtype=torch.uint8, device=x.device)
    args = _NormArgs(b, p, c, g, TYPES[x.dtype], ACTS[act], eps, ptr, ld, mk, gm, bt, stats.data_ptr(),
                     stats.data_ptr() + 4 * b * g, work.data_ptr(), yp, ldy, None, 0, None, 0, None, None)
    _check(L.kg_group_norm(x.device.index, _stream(x.device), ctypes.byref(args)))
    return y, stats[0], stats[1]


def group_norm_backward(dy, x, mean, rstd, groups, gamma=None, beta=None, *, mask=None, act="identity", dx=None):
    """The gradients (dx, dgamma, dbeta) of a loss whose gradient with respect to group_norm's y is dy, from its mean and rstd
    (kg_group_norm_backward); dx into `dx` when given."""
    ptr, ld = _points(x, "x")
    b, p, c, g, mk, gm, bt = _norm_shape(x, groups, gamma, beta, mask, act)
    dev = x.device
    if dx is None:
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    for t, name in ((dy, "dy"), (dx, "dx")):
        if t.shape != x.shape or t.dtype != x.dtype or t.device != dev:
            raise ValueError(f"{name} must have the shape, type and device of x")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.shape != (b, g) or t.dtype != torch.float32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape ({b}, {g}) on {dev}")
    dyp, lddy = _points(dy, "dy")
    dxp, lddx = _points(dx, "dx")
    L = _library()
    out = torch.empty(2, c, dtype=torch.float32, device=dev)
    work = torch.empty(L.kg_group_norm_workspace(b, p, c, g, 1), dtype=torch.uint8, device=dev)
    args = _NormArgs(b, p, c, g, TYPES[x.dtype], ACTS[act], 0.0, ptr, ld, mk, gm, bt, mean.data_ptr(), rstd.data_ptr(),
                     work.data_ptr(), None, 0, dyp, lddy, dxp, lddx, out.data_ptr(), out.data_ptr() + 4 * c)
    _check(L.kg_group_norm_backward(dev.index, _stream(dev), ctypes.byref(args)))
    return dx, out[0], out[1]


class AdamW:
    """AdamW over a list of parameters, one call a step (kg_adamw_step). The parameters (contiguous float32, float16 or
    bfloat16 tensors of one GPU) and their float32 `masters` (a list, None where a parameter has none) are updated in place.
    weight_decay is one number or one for each parameter. The moments of all parameters lie in one state (m, v and, in 8 bits,
    m_exp, v_exp), each parameter's from element BLOCK * first_block[i] on; a program saves state() and gives it to load_state."""

    def __init__(self, params, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, masters=None):
        params = list(params)
        masters = [None] * len(params) if masters is None else list(masters)
        decays = list(weight_decay) if hasattr(weight_decay, "__len__") else [weight_decay] * len(params)
        if not params:
            raise ValueError("AdamW needs a parameter")
        if len(masters) != len(params) or len(decays) != len(params):
            raise ValueError(f"AdamW needs {len(params)} masters and weight decays")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.device = params[0].device
        for i, (p, w) in enumerate(zip(params, masters)):
            if p.dtype not in TYPES or not p.is_cuda or p.device != self.device or not p.is_contiguous():
                raise ValueError(f"parameter {i} must be contiguous float32, float16 or bfloat16 on one GPU")
            if w is not None and (w.dtype != torch.float32 or w.shape != p.shape or w.device != self.device or
                                  not w.is_contiguous()):
                raise ValueError(f"master {i} must be contiguous float32 of its parameter's shape and device")
        self.params, self.masters, self.state_bits = params, masters, state_bits
        self.lr, self.betas, self.eps = lr, tuple(betas), eps
        self.step_count = 0
        blocks = [-(-p.numel() // BLOCK) for p in params]
        self.first_block = np.concatenate([[0], np.cumsum(blocks)]).astype(np.int64)
        total = int(self.first_block[-1])
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.m = torch.zeros(total * BLOCK, dtype=kind, device=self.device)
        self.v = torch.zeros(total * BLOCK, dtype=kind, device=self.device)
        exps = [None, None] if state_bits == 32 else [torch.zeros(total, dtype=torch.uint8, device=self.device)
                                                      for _ in range(2)]
        self.m_exp, self.v_exp = exps
        self._state = _AdamState(state_bits, *(None if t is None else t.data_ptr() for t in (self.m, self.v, *exps)))
        self._tensors = (_AdamTensor * len(params))()
        self._rec = np.frombuffer(self._tensors, np.dtype(_AdamTensor))
        self._rec["param"] = [p.data_ptr() for p in params]
        self._rec["master"] = [0 if w is None else w.data_ptr() for w in masters]
        self._rec["first_block"] = self.first_block[:-1]
        self._rec["weight_decay"] = decays
        self._rec["param_type"] = [TYPES[p.dtype] for p in params]
        self.grads = None

    def bind(self, grads):
        """Takes the gradients that the next steps read: one contiguous tensor a parameter, or None where it has none (it
        is left as it is). A program whose gradients stay in place binds them once."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"AdamW needs {len(self.params)} gradients, got {len(grads)}")
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is not None and (g.dtype not in TYPES or g.shape != p.shape or g.device != self.device or
                                  not g.is_contiguous()):
                raise ValueError(f"gradient {i} must be contiguous float32, float16 or bfloat16 of its parameter's shape "
                                 "and device")
        self._rec["grad"] = [0 if g is None else g.data_ptr() for g in grads]
        self._rec["grad_type"] = [0 if g is None else TYPES[g.dtype] for g in grads]
        self._rec["elements"] = [0 if g is None else g.numel() for g in grads]
        self.grads = grads

    def _hyper(self, lr, step, grad_scale, seed):
        return _AdamHyper(self.lr if lr is None else lr, *self.betas, self.eps, grad_scale, step,
                          (step if seed is None else seed) & 0xFFFFFFFF)

    def step(self, grads=None, *, lr=None, step=None, grad_scale=1.0, seed=None, values=None):
        """One step with `grads` (or the bound ones). step: its number, from 1 (the next one by default); seed: of the 8-bit
        moments' rounding (the step's number by default); values: a device tensor that holds an AdamValues, read by the kernel
        in place of these numbers, for a step that is captured once and replayed."""
        if grads is not None:
            self.bind(grads)
        if self.grads is None:
            raise ValueError("AdamW.step needs gradients: give or bind them")
        if values is not None and (not values.is_cuda or values.device != self.device or not values.is_contiguous() or
                                   values.numel() * values.element_size() < ctypes.sizeof(AdamValues)):
            raise ValueError(f"values must be {ctypes.sizeof(AdamValues)} bytes on {self.device}")
        number = self.step_count + 1 if step is None else step
        _check(_library().kg_adamw_step(self.device.index, _stream(self.device), len(self.params),
                                        ctypes.byref(self._tensors), ctypes.byref(self._state),
                                        ctypes.byref(self._hyper(lr, number, grad_scale, seed)), None if values is None else values.data_ptr()))
        self.step_count = number

    def values(self, *, lr=None, step=None, grad_scale=1.0, seed=None):
        """The scalars of a step (the next one by default) as a uint8 tensor on the host, to be copied to a captured step's
        `values`."""
        out = AdamValues()
        number = self.step_count + 1 if step is None else step
        _check(lib().kg_adamw_values(ctypes.byref(self._hyper(lr, number, grad_scale, seed)), ctypes.byref(out)))
        return torch.frombuffer(bytearray(out), dtype=torch.uint8)

    def moments(self, dtype=None):
        """The moments as numbers, in the state's layout: m and sqrt(v) (8 bits: bfloat16 by default, which holds them
        exactly; 32 bits: float32)."""
        dtype = dtype or (torch.float32 if self.state_bits == 32 else torch.bfloat16)
        if dtype not in TYPES:
            raise ValueError("moments are given as float32, float16 or bfloat16")
        m, root = (torch.empty(self.m.numel(), dtype=dtype, device=self.device) for _ in range(2))
        _check(_library().kg_adamw_moments(self.device.index, _stream(self.device), self.m.numel() // BLOCK,
                                           ctypes.byref(self._state),
                                           TYPES[dtype], m.data_ptr(), root.data_ptr()))
        return m, root

    def state(self):
        """The optimizer's state: the tensors of load_state, and the number of steps taken."""
        names = ("m", "v") if self.state_bits == 32 else ("m", "v", "m_exp", "v_exp")
        return {k: getattr(self, k) for k in names}, self.step_count

    def load_state(self, tensors, step_count):
        """Copies the tensors of a state (m and v, in 8 bits also m_exp and v_exp) and its number of steps."""
        names = ("m", "v") if self.state_bits == 32 else ("m", "v", "m_exp", "v_exp")
        for k in names:
            own = getattr(self, k)
            if k not in tensors or tensors[k].shape != own.shape or tensors[k].dtype != own.dtype:
                raise ValueError(f"the state's {k} must be {own.numel()} {str(own.dtype)[6:]}")
        for k in names:
            getattr(self, k).copy_(tensors[k])
        self.step_count = int(step_count)
