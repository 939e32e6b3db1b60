"""The learning operators' argument structures as a C caller declares them (include/kgx.h)."""

import ctypes

_vp, _ci, _ll, _cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double


class PolicyArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("columns", _ci), ("type", _ci), ("logits", _vp), ("ld", _ll), ("legal", _vp),
                ("ld_legal", _ll), ("action", _vp), ("old_logp", _vp), ("advantage", _vp), ("weight", _vp),
                ("ref_logits", _vp), ("ld_ref", _ll), ("ref_logp", _vp), ("logit_scale", _cd), ("clip_low", _cd),
                ("clip_high", _cd), ("kl_coef", _cd), ("loss", _vp), ("logp", _vp), ("kl", _vp), ("grad", _vp),
                ("ld_grad", _ll), ("workspace", _vp)]


class PreferenceArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("columns", _ci), ("type", _ci), ("logits", _vp), ("ld", _ll), ("label", _vp),
                ("pairs", _ci), ("offsets", _vp), ("ref_logp", _vp), ("weight", _vp), ("beta", _cd),
                ("label_smoothing", _cd), ("average", _ci), ("loss", _vp), ("margin", _vp), ("seq_logp", _vp),
                ("grad", _vp), ("ld_grad", _ll), ("workspace", _vp)]


class NormArgs(ctypes.Structure):
    _fields_ = [("batch", _ci), ("points", _ci), ("channels", _ci), ("groups", _ci), ("type", _ci), ("act", _ci),
                ("eps", _cd), ("x", _vp), ("ldx", _ll), ("mask", _vp), ("gamma", _vp), ("beta", _vp), ("mean", _vp),
                ("rstd", _vp), ("workspace", _vp), ("y", _vp), ("ldy", _ll), ("dy", _vp), ("lddy", _ll), ("dx", _vp),
                ("lddx", _ll), ("dgamma", _vp), ("dbeta", _vp)]
