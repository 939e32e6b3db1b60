"""The argument structures of a student's operators as a C caller declares them (include/kgx.h)."""

import ctypes

_vp, _ci, _ll, _cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double


class DistillArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("columns", _ci), ("k", _ci), ("type", _ci), ("top_type", _ci), ("logits", _vp), ("ld", _ll),
                ("legal", _vp), ("ld_legal", _ll), ("top_index", _vp), ("ld_index", _ll), ("top_logits", _vp), ("ld_top", _ll),
                ("teacher_lse", _vp), ("weight", _vp), ("logit_scale", _cd), ("loss", _vp), ("grad", _vp), ("ld_grad", _ll),
                ("workspace", _vp)]


class LayerArgs(ctypes.Structure):
    _fields_ = [("rows", _ci), ("channels", _ci), ("type", _ci), ("rms", _ci), ("eps", _cd), ("x", _vp), ("ldx", _ll),
                ("gamma", _vp), ("beta", _vp), ("mean", _vp), ("rstd", _vp), ("workspace", _vp), ("y", _vp), ("ldy", _ll),
                ("dy", _vp), ("lddy", _ll), ("dx", _vp), ("lddx", _ll), ("dgamma", _vp), ("dbeta", _vp)]


class EmbedArgs(ctypes.Structure):
    _fields_ = [("count", _ci), ("vocab", _ci), ("channels", _ci), ("type", _ci), ("tokens", _vp), ("scale", _cd), ("table", _vp),
                ("ld_table", _ll), ("y", _vp), ("ld_y", _ll), ("dy", _vp), ("ld_dy", _ll), ("grad_type", _ci),
                ("accumulate", _ci), ("grad", _vp), ("ld_grad", _ll), ("workspace", _vp)]
