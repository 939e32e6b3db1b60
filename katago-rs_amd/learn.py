"""Learning from the network's answers: the operators of include/kgx.h's last section on torch tensors of a GPU.

- `policy_loss`: the clipped policy loss with a KL term on rows of logits (a network's policy rows with their legal moves,
  or tokens), and its gradient;
- `preference_loss`: pairs of lines of moves or token sequences, the better against the worse, and its gradient;
- `AdamW`: one step over many tensors at once, moments in 32 or in 8 bits;
- `group_norm` and `group_norm_backward`: group norm with an activation on channels-last rows under the board mask.

The calls run on torch's current stream of the tensors' device and do not wait. They take part in no autograd graph: gradients
are returned. What they write into a caller's tensor raises its version counter as torch's own in-place operations do (a replayed
graph raises none, as with those). There is no other compute path, and a call that the library refuses raises KgError; a tensor of another shape,
type or device than the call needs, or a size past 31 bits, raises ValueError. A network's own policy rows come from Handle.policy_rows:

    rows = torch.as_tensor(handle.policy_rows(n), device="cuda")   # [n, 362], inside the raw rows
    r = learn.policy_loss(rows, actions, old_logp, advantage, legal=legal, kl_coef=0.1, ref_logits=before)

torch has to be imported before the library is loaded (importing this module first does that): both use the process's one HIP
runtime.
"""

import collections
import ctypes
import math
import operator
import struct

import numpy as np
import torch

from . import KgError, PRECISION_BF16, PRECISION_F16, PRECISION_F32, _check, lib

TYPES = {torch.float32: PRECISION_F32, torch.float16: PRECISION_F16, torch.bfloat16: PRECISION_BF16}
ACTS = {"identity": 0, "relu": 1, "mish": 2, "silu": 3}
BLOCK = 256  # KG_ADAMW_BLOCK
_BYTES = (torch.bool, torch.uint8)
_DTYPE, _DEVICE = operator.attrgetter("dtype"), torch.Tensor.get_device
_NUMEL, _CONTIGUOUS, _POINTER = torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.data_ptr

PolicyLoss = collections.namedtuple("PolicyLoss", ["loss", "logp", "kl", "grad"])
PreferenceLoss = collections.namedtuple("PreferenceLoss", ["loss", "margin", "seq_logp", "grad"])

_vp, _ci, _ll, _cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double


# The argument structures of include/kgx.h, packed at their natural alignment: a third of a ctypes structure's time, and a small
# batch's call is its host time. (A size past 31 bits does not pack: _out_of_range.)
_POLICY_ARGS = struct.Struct("@3iPqPqPPPPPqPddddPPPPqP0q")
_PREFERENCE_ARGS = struct.Struct("@3iPqPiPPPddiPPPPqP0q")
_NORM_ARGS = struct.Struct("@6idPqPPPPPPPqPqPqPP0q")


def _out_of_range(op, error):
    return ValueError(f"{op}: a size or number is out of range ({error})")


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


# The handle of torch's current stream of a device, without the Stream object around it where torch offers that.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _rows(t, name, like=None):
    """(pointer, row stride) of a matrix on the GPU with unit column stride; `like`: of that shape, type and device."""
    ld = t.stride()
    if len(ld) != 2 or t.dtype not in TYPES or (ld[1] != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be [rows, columns] of float32, float16 or bfloat16 with contiguous columns")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if like is not None and (t.shape != like.shape or t.dtype is not like.dtype or t.get_device() != like.get_device()):
        raise ValueError(f"{name} must have the shape, type and device of the logits")
    return t.data_ptr(), ld[0]


def _vector(t, n, dtype, name, device):
    """Pointer of a contiguous vector of n elements on GPU number `device`; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} {str(dtype)[6:]} on GPU {device}")
    return t.data_ptr()


_written = torch.autograd.graph.increment_version


def _workspace(size, device):
    """A call's workspace, None for 0 bytes. The caller holds it until the library has been called: memory that goes back to the
    allocator before that is another thread's to take, with kernels of its own between this call's."""
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def policy_loss(logits, actions, old_logp, advantage, *, legal=None, weight=None, logit_scale=1.0, clip=(0.2, 0.2),
                kl_coef=0.0, ref_logits=None, ref_logp=None, want_grad=True, grad=None):
    """The clipped policy loss of each row with its KL term, and the gradient of their sum (kg_policy_loss).

    logits [n, v] (rows may be strided); actions [n] int32, outside [0, v) for padding; old_logp, advantage, weight [n]
    float32; legal [n, v] bool or uint8; clip (low, high): the ratio counts within [1 - low, 1 + high]; the KL term is the full
    one to ref_logits [n, v], or the estimate from ref_logp [n]. Returns loss, logp and kl [n] float32 and grad [n, v] of
    the logits' type (into `grad` when given; None without want_grad)."""
    ptr, ld = _rows(logits, "logits")
    n, v = logits.shape
    dev = logits.get_device()
    lg = ld_lg = ref = ld_ref = g = ld_g = 0
    if legal is not None:
        if legal.shape != (n, v) or legal.dtype not in _BYTES or legal.get_device() != dev or (legal.stride(1) != 1 and v > 1):
            raise ValueError(f"legal must be [{n}, {v}] bool or uint8 on GPU {dev} with contiguous columns")
        lg, ld_lg = legal.data_ptr(), legal.stride(0)
    if ref_logits is not None:
        ref, ld_ref = _rows(ref_logits, "ref_logits", logits)
    given = grad
    if grad is not None:
        g, ld_g = _rows(grad, "grad", logits)
    elif want_grad:
        grad = torch.empty((n, v), dtype=logits.dtype, device=logits.device)
        g, ld_g = grad.data_ptr(), v
    loss, logp, kl = torch.empty((3, n), dtype=torch.float32, device=logits.device).unbind()
    o = loss.data_ptr()
    L = _library()
    # (Few long rows: 16384 columns are the least that a workspace is for.)
    bytes_ = L.kg_policy_loss_workspace(n, v) if v > 16384 else 0
    work = _workspace(bytes_, logits.device)
    try:
        args = _POLICY_ARGS.pack(n, v, TYPES[logits.dtype], ptr, ld, lg, ld_lg, _vector(actions, n, torch.int32, "actions", dev),
                                 _vector(old_logp, n, torch.float32, "old_logp", dev),
                                 _vector(advantage, n, torch.float32, "advantage", dev),
                                 _vector(weight, n, torch.float32, "weight", dev), ref, ld_ref,
                                 _vector(ref_logp, n, torch.float32, "ref_logp", dev), logit_scale, clip[0], clip[1], kl_coef, o,
                                 o + 4 * n, o + 8 * n, g, ld_g, work.data_ptr() if work is not None else 0)
    except struct.error as e:
        raise _out_of_range("policy_loss", e) from None
    if L.kg_policy_loss(dev, _stream(dev), args):
        _check(1)
    if given is not None:
        _written(given)
    return PolicyLoss(loss, logp, kl, grad)


def preference_loss(logits, labels, offsets, ref_logp, *, beta=0.1, label_smoothing=0.0, average=False, weight=None,
                    want_grad=True, grad=None):
    """The preference loss of pairs of sequences packed in rows of logits, and the gradient of its sum (kg_preference_loss).

    logits [t, v] (rows may be strided); labels [t] int32, outside [0, v) where a row is not counted; offsets [2 p + 1] int32:
    sequence q is rows [offsets[q], offsets[q + 1]), and pair i prefers sequence 2 i to 2 i + 1; ref_logp [2 p] float32: the
    sequences' log-probabilities (means with `average`) under the reference; weight [p] float32. Returns loss and margin [p],
    seq_logp [2 p] and grad [t, v] of the logits' type (into `grad` when given; None without want_grad)."""
    ptr, ld = _rows(logits, "logits")
    t, v = logits.shape
    dev = logits.get_device()
    g = ld_g = 0
    if offsets.dim() != 1 or offsets.shape[0] % 2 == 0:
        raise ValueError("offsets must be a vector of an odd length")
    p = offsets.shape[0] // 2
    given = grad
    if grad is not None:
        g, ld_g = _rows(grad, "grad", logits)
    elif want_grad:
        grad = torch.empty((t, v), dtype=logits.dtype, device=logits.device)
        g, ld_g = grad.data_ptr(), v
    L = _library()
    # (One allocation: the pairs' results, then the workspace at a multiple of 256 bytes.)
    room = -(-16 * p // 256) * 256
    out = torch.empty(room // 4 + L.kg_preference_loss_workspace(t) // 4, dtype=torch.float32, device=logits.device)
    loss, margin, seq_logp, _ = out.split_with_sizes((p, p, 2 * p, out.numel() - 4 * p))
    o = out.data_ptr()
    try:
        args = _PREFERENCE_ARGS.pack(t, v, TYPES[logits.dtype], ptr, ld, _vector(labels, t, torch.int32, "labels", dev), p,
                                     _vector(offsets, 2 * p + 1, torch.int32, "offsets", dev),
                                     _vector(ref_logp, 2 * p, torch.float32, "ref_logp", dev),
                                     _vector(weight, p, torch.float32, "weight", dev), beta, label_smoothing, bool(average), o,
                                     o + 4 * p, o + 8 * p, g, ld_g, o + room)
    except struct.error as e:
        raise _out_of_range("preference_loss", e) from None
    if L.kg_preference_loss(dev, _stream(dev), args):
        _check(1)
    if given is not None:
        _written(given)
    return PreferenceLoss(loss, margin, seq_logp, grad)


def _points(t, name):
    """(pointer, row stride) of [batch, ..., channels] whose points lie evenly spaced."""
    shape = t.shape
    if len(shape) < 2 or t.dtype not in TYPES:
        raise ValueError(f"{name} must be [batch, ..., channels] of float32, float16 or bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if t.is_contiguous() or not t.numel():
        return t.data_ptr(), shape[-1]
    ld = None
    span = 1
    for size, stride in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
        if size != 1:
            if ld is None:
                ld = stride
            elif stride != ld * span:
                raise ValueError(f"the points of {name} must be evenly spaced")
            span *= size
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous channels")
    return t.data_ptr(), shape[-1] if ld is None else ld


def _norm_shape(x, groups, gamma, beta, mask, act):
    shape, dev = x.shape, x.get_device()
    if act not in ACTS:
        raise ValueError(f"act must be one of {', '.join(ACTS)}")
    batch, channels = shape[0], shape[-1]
    points = shape[1] if len(shape) == 3 else math.prod(shape[1:-1])
    mk = 0
    if mask is not None:
        if mask.dtype is not torch.float32 or mask.shape != shape[:-1] or mask.get_device() != dev or not mask.is_contiguous():
            raise ValueError(f"mask must be contiguous float32 of shape {tuple(shape[:-1])} on GPU {dev}")
        mk = mask.data_ptr()
    return (dev, batch, points, channels, int(groups), mk, _vector(gamma, channels, torch.float32, "gamma", dev),
            _vector(beta, channels, torch.float32, "beta", dev))


def _like(t, x, name):
    if t.shape != x.shape or t.dtype is not x.dtype or t.get_device() != x.get_device():
        raise ValueError(f"{name} must have the shape, type and device of x")
    return _points(t, name)


def group_norm(x, groups, gamma=None, beta=None, *, mask=None, eps=1e-5, act="identity", y=None):
    """act(group norm of x) on channels-last x [batch, ..., channels] over the points with a nonzero mask [batch, ...]
    (kg_group_norm). Returns y (into `y` when given; 0 where the mask is 0), and mean and rstd [batch, groups]."""
    ptr, ld = _points(x, "x")
    dev, b, p, c, g, mk, gm, bt = _norm_shape(x, groups, gamma, beta, mask, act)
    given = y
    if y is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        yp, ldy = y.data_ptr(), c
    else:
        yp, ldy = _like(y, x, "y")
    L = _library()
    stats = torch.empty((2, b, max(min(g, c), 0)), dtype=torch.float32, device=x.device)
    work = _workspace(L.kg_group_norm_workspace(b, p, c, g, 0), x.device)
    mean, rstd = stats.unbind()
    o = stats.data_ptr()
    try:
        args = _NORM_ARGS.pack(b, p, c, g, TYPES[x.dtype], ACTS[act], eps, ptr, ld, mk, gm, bt, o, o + 4 * b * g,
                               work.data_ptr() if work is not None else 0, yp, ldy, 0, 0, 0, 0, 0, 0)
    except struct.error as e:
        raise _out_of_range("group_norm", e) from None
    if L.kg_group_norm(dev, _stream(dev), args):
        _check(1)
    if given is not None:
        _written(given)
    return y, mean, rstd


def group_norm_backward(dy, x, mean, rstd, groups, gamma=None, beta=None, *, mask=None, act="identity", dx=None):
    """The gradients (dx, dgamma, dbeta) of a loss whose gradient with respect to group_norm's y is dy, from its mean and rstd
    (kg_group_norm_backward); dx into `dx` when given."""
    ptr, ld = _points(x, "x")
    dev, b, p, c, g, mk, gm, bt = _norm_shape(x, groups, gamma, beta, mask, act)
    dyp, lddy = _like(dy, x, "dy")
    given = dx
    if dx is None:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dxp, lddx = dx.data_ptr(), c
    else:
        dxp, lddx = _like(dx, x, "dx")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype is not torch.float32 or t.shape != (b, g) or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape ({b}, {g}) on GPU {dev}")
    L = _library()
    work = _workspace(L.kg_group_norm_workspace(b, p, c, g, 1), x.device)
    out = torch.empty((2, c), dtype=torch.float32, device=x.device)
    dgamma, dbeta = out.unbind()
    o = out.data_ptr()
    try:
        args = _NORM_ARGS.pack(b, p, c, g, TYPES[x.dtype], ACTS[act], 0.0, ptr, ld, mk, gm, bt, mean.data_ptr(), rstd.data_ptr(),
                               work.data_ptr() if work is not None else 0, 0, 0, dyp, lddy, dxp, lddx, o, o + 4 * c)
    except struct.error as e:
        raise _out_of_range("group_norm_backward", e) from None
    if L.kg_group_norm_backward(dev, _stream(dev), args):
        _check(1)
    if given is not None:
        _written(given)
    return dx, dgamma, dbeta


class AdamW:
    """AdamW over a list of parameters, one call a step (kg_adamw_step). The parameters (contiguous float32, float16 or
    bfloat16 tensors of one GPU) and their float32 `masters` (a list, None where a parameter has none) are updated in place,
    where they lie now.
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
        places = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                        for t in (*params, *masters) if t is not None and t.numel())
        if any(end > start for (_, end), (start, _) in zip(places, places[1:])):
            raise ValueError("each parameter and master must be a tensor of its own that shares no memory with another")
        self.params, self.masters, self.state_bits = params, masters, state_bits
        # One tensor a version counter, which views share with their base: raising 400 takes 19 us.
        bases = (t if t._base is None else t._base for t in (*params, *masters) if t is not None)
        self._counters = list({id(t): t for t in bases}.values())
        self.lr, self.betas, self.eps = lr, tuple(betas), eps
        self.step_count = 0
        self._sizes = [p.numel() for p in params]
        self._elements = np.array(self._sizes, np.int64)
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
        # (Whole lists at once: a network has hundreds of gradients, and a step's time on the GPU is near this one's.)
        try:
            kinds = self._check_grads(grads, self._sizes)
            some, here, sizes = grads, slice(None), self._elements
        except TypeError:  # (None has no sizes)
            here = [g is not None for g in grads]
            some = [g for g in grads if g is not None]
            sizes = self._elements[here]
            kinds = self._check_grads(some, sizes.tolist())
            self._rec["grad"] = self._rec["grad_type"] = self._rec["elements"] = 0
        self._rec["grad"][here] = list(map(_POINTER, some))
        self._rec["grad_type"][here] = kinds
        self._rec["elements"][here] = sizes
        self.grads = grads

    def _check_grads(self, grads, sizes):
        own = list(map(_NUMEL, grads))
        types = list(map(_DTYPE, grads))
        if own != sizes or not all(map(_CONTIGUOUS, grads)) or \
                set(map(_DEVICE, grads)) - {self.device.index} or set(types) - TYPES.keys():
            raise ValueError("each gradient must be contiguous float32, float16 or bfloat16 of its parameter's size and GPU")
        return TYPES[types[0]] if len(set(types)) == 1 else [TYPES[t] for t in types]

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
        dev = self.device.index
        _check(_library().kg_adamw_step(dev, _stream(dev), len(self.params),
                                        ctypes.byref(self._tensors), ctypes.byref(self._state),
                                        ctypes.byref(self._hyper(lr, number, grad_scale, seed)), None if values is None else values.data_ptr()))
        _written(self._counters)
        self.step_count = number

    def values(self, *, lr=None, step=None, grad_scale=1.0, seed=None):
        """The scalars of a step (the next one by default) as a uint8 tensor on the host, to be copied to a captured step's
        `values`. Replays are not counted: a program that replays gives `step`."""
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
        m, root = torch.empty((2, self.m.numel()), dtype=dtype, device=self.device).unbind()
        _check(_library().kg_adamw_moments(self.device.index, _stream(self.device.index), self.m.numel() // BLOCK,
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
