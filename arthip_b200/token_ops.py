"""Token operators on device tensors (``ah_norm_*``, ``ah_rope_*``, ``ah_attn_*``): the layers
that stand between conv layers in attention-based restoration models. A token is a pixel or a
patch of a frame, so a conv layer's NHWC frame is ``[tokens][channels]`` as it stands.

* :class:`TokenNorm`: the norms before and after a block with its gate and residual scale.
* :class:`AxisRotary`: rotary positions over time, height and width.
* :class:`TokenAttention`: attention with a score cap, distance biases, documents, causal and
  prefix masks, for whole frames and for single new tokens against a cache.

Tensors are given as device pointers (ints), as to :class:`~arthip_b200.engine.Conv3x3`;
strides count elements and 0 means packed. Element types are "fp16" and "bf16". A handle may
run on several streams and threads at once, and runs may be captured into CUDA graphs.
"""

from __future__ import annotations

import ctypes

import numpy as np

from .engine import EngineHarnessError, _ERR_LEN, _err, _msg
from .native import lib

_i32, _i64, _f32, _f64, _vp = (ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_void_p)
_DTYPES = {"fp16": 0, "bf16": 1}
_NORMS = {"none": 0, "rms": 1, "layer": 2}
_GATES = {"none": 0, "sigmoid": 1, "tanh": 2, "silu": 3}
_LAYOUTS = {"halves": 0, "pairs": 1, "shared": 2}
_MASKS = {"full": 0, "causal": 1}
_ALGOS = {"auto": 0, "mma": 1, "tc": 2}


class _NormDesc(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("channels", _i32), ("post_norm", _i32), ("pre_norm", _i32), ("post_eps", _f32),
                ("pre_eps", _f32), ("gate_act", _i32), ("residual_scale", _f32)]


class _NormIo(ctypes.Structure):
    _fields_ = [("rows", _i64), ("x", _vp), ("y", _vp), ("gate", _vp), ("mod_scale", _vp), ("mod_shift", _vp),
                ("out", _vp), ("norm", _vp), ("x_stride", _i64), ("y_stride", _i64), ("gate_stride", _i64),
                ("mod_stride", _i64), ("out_stride", _i64), ("norm_stride", _i64), ("rows_per_gate", _i64),
                ("rows_per_mod", _i64)]


class _RopeDesc(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("head_dim", _i32), ("axes", _i32), ("axis_dims", _i32 * 3), ("theta", _f64 * 3),
                ("layout", _i32), ("inverse", _i32)]


class _RopeIo(ctypes.Structure):
    _fields_ = [("in_", _vp), ("out", _vp), ("heads", _i32), ("in_token_stride", _i64), ("in_head_stride", _i64),
                ("out_token_stride", _i64), ("out_head_stride", _i64)]


class _AttnDesc(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("q_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("scale", _f32),
                ("cap", _f32), ("mask", _i32), ("axes", _i32), ("algo", _i32)]


class _AttnIo(ctypes.Structure):
    _fields_ = [("q", _vp), ("k", _vp), ("v", _vp), ("out", _vp), ("q_token_stride", _i64), ("q_head_stride", _i64),
                ("k_token_stride", _i64), ("k_head_stride", _i64), ("v_token_stride", _i64), ("v_head_stride", _i64),
                ("out_token_stride", _i64), ("out_head_stride", _i64), ("q_positions", _vp), ("k_positions", _vp),
                ("k_lens", _vp)]


def _code(table: dict, value: str, what: str) -> int:
    if value not in table:
        raise EngineHarnessError(f"unknown {what} {value!r} (one of {', '.join(table)})")
    return table[value]


def _floats(v, shape, what: str):
    """A host fp32 array of this shape, or None."""
    if v is None:
        return None
    v = np.ascontiguousarray(v, dtype=np.float32)
    if v.shape != shape:
        raise EngineHarnessError(f"{what} has shape {v.shape}, not {shape}")
    return v


def _whole(v, what: str):
    """A host int64 array of one dimension, from whole numbers only."""
    v = np.asarray(v)
    if v.ndim != 1 or (v.size and not np.issubdtype(v.dtype, np.integer)):
        raise EngineHarnessError(f"{what} must be a list of whole numbers")
    return np.ascontiguousarray(v, dtype=np.int64)


def _data(v):
    return None if v is None else v.ctypes.data


class _Handle:
    _destroy = ""

    def __init__(self):
        self._lib = lib()
        self._h = ctypes.c_void_p()

    def _check(self, rc: int, err, what: str):
        if rc != 0:
            raise EngineHarnessError(_msg(err, f"{what} failed (rc={rc})"))

    def close(self):
        """Frees the handle; its runs must have finished."""
        if self._h:
            getattr(self._lib, self._destroy)(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class TokenNorm(_Handle):
    """``out = x + residual_scale * layer_scale * act(gate) * post(y)`` and
    ``norm = pre(out) * (1 + mod_scale) + mod_shift``, in one pass over the rows.

    ``post_norm`` / ``pre_norm``: "none", "rms" or "layer"; weights, biases and layer scale
    are host arrays of ``channels`` floats. ``gate_act``: "none" (the gate as it is),
    "sigmoid", "tanh" or "silu"."""

    _destroy = "ah_norm_destroy"

    def __init__(self, channels: int, dtype: str = "fp16", post_norm: str = "none", pre_norm: str = "rms",
                 post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, layer_scale=None,
                 gate_act: str = "none", residual_scale: float = 1.0, post_eps: float = 1e-6, pre_eps: float = 1e-6,
                 device: int = 0):
        super().__init__()
        d = _NormDesc(_code(_DTYPES, dtype, "dtype"), channels, _code(_NORMS, post_norm, "norm"),
                      _code(_NORMS, pre_norm, "norm"), post_eps, pre_eps, _code(_GATES, gate_act, "gate activation"),
                      residual_scale)
        w = [_floats(v, (channels,), name) for v, name in (
            (post_weight, "post_weight"), (post_bias, "post_bias"), (pre_weight, "pre_weight"),
            (pre_bias, "pre_bias"), (layer_scale, "layer_scale"))]
        err = _err()
        self._check(self._lib.ah_norm_create(device, ctypes.byref(d), *map(_data, w), ctypes.byref(self._h), err,
                                             _ERR_LEN), err, "norm create")
        self.channels = channels

    def run(self, rows: int, x_ptr: int, out_ptr: int = 0, norm_ptr: int = 0, y_ptr: int = 0, gate_ptr: int = 0,
            rows_per_gate: int = 1, mod_scale_ptr: int = 0, mod_shift_ptr: int = 0, rows_per_mod: int = 1,
            x_stride: int = 0, y_stride: int = 0, gate_stride: int = 0, mod_stride: int = 0, out_stride: int = 0,
            norm_stride: int = 0, stream: int = 0):
        """Row r uses gate row ``r // rows_per_gate`` and modulation row ``r // rows_per_mod``.
        Without ``y_ptr`` only the pre-norm of x is taken."""
        io = _NormIo(rows, x_ptr, y_ptr, gate_ptr, mod_scale_ptr, mod_shift_ptr, out_ptr, norm_ptr, x_stride, y_stride,
                     gate_stride, mod_stride, out_stride, norm_stride, rows_per_gate, rows_per_mod)
        err = _err()
        self._check(self._lib.ah_norm_run(self._h, ctypes.byref(io), stream or None, err, _ERR_LEN), err, "norm run")


class AxisRotary(_Handle):
    """Rotary positions: ``axis_dims[i]`` (even) elements of each head turn with axis i.

    ``layout``: "halves" (pair j of a section is its elements j and j + half), "pairs"
    (elements 2j and 2j + 1) or "shared" (one spectrum over the whole rotated part, its
    pairs shared out over the axes). ``theta``: one base or one per axis. ``inverse`` turns
    the other way."""

    _destroy = "ah_rope_destroy"

    def __init__(self, head_dim: int, axis_dims, theta=10000.0, layout: str = "halves", dtype: str = "fp16",
                 inverse: bool = False, device: int = 0):
        super().__init__()
        dims = [int(n) for n in axis_dims]
        thetas = [float(theta)] * len(dims) if np.isscalar(theta) else [float(t) for t in theta]
        if not 1 <= len(dims) <= 3 or len(thetas) != len(dims):
            raise EngineHarnessError("axis_dims names 1 to 3 axes, theta one base or one for each")
        d = _RopeDesc(_code(_DTYPES, dtype, "dtype"), head_dim, len(dims), (_i32 * 3)(*dims), (_f64 * 3)(*thetas),
                      _code(_LAYOUTS, layout, "layout"), int(inverse))
        err = _err()
        self._check(self._lib.ah_rope_create(device, ctypes.byref(d), ctypes.byref(self._h), err, _ERR_LEN), err,
                    "rope create")
        self.head_dim, self.axes = head_dim, len(dims)

    def run(self, tokens: int, positions_ptr: int, q_ptr: int, q_heads: int, q_out_ptr: int = 0, k_ptr: int = 0,
            k_heads: int = 0, k_out_ptr: int = 0, q_strides=(0, 0), k_strides=(0, 0), q_out_strides=None,
            k_out_strides=None, stream: int = 0):
        """``positions_ptr``: fp32 [axes][tokens]. Strides are (token, head); an output pointer
        of 0 turns in place, with the input's strides; outputs of their own are packed unless
        strides are given. ``k_ptr`` 0: q alone."""
        def io(src, heads, dst, strides, out_strides):
            out = out_strides if out_strides is not None else ((0, 0) if dst else strides)
            return _RopeIo(src, dst or src, heads, *strides, *out)
        q = io(q_ptr, q_heads, q_out_ptr, q_strides, q_out_strides) if q_ptr else None
        k = io(k_ptr, k_heads, k_out_ptr, k_strides, k_out_strides) if k_ptr else None
        err = _err()
        self._check(self._lib.ah_rope_run(self._h, tokens, positions_ptr or None, q and ctypes.byref(q),
                                          k and ctypes.byref(k), stream or None, err, _ERR_LEN), err, "rope run")


class TokenAttention(_Handle):
    """Attention over documents packed one after another: queries ``q_offsets[i]`` to
    ``q_offsets[i + 1]`` see the keys ``k_offsets[i]`` to ``k_offsets[i + 1]``.

    ``mask``: "full", or "causal" (aligned to the last key), with ``prefix[i]`` first keys that
    every query of document i sees. ``cap``: scores become ``cap * tanh(score / cap)``.
    ``slopes`` [q_heads][axes]: ``slope * |q position - k position|`` is taken off the scores
    for each axis. The softmax weights are rounded to ``dtype`` before they multiply the values;
    scores and sums are fp32. ``scale`` defaults to ``head_dim ** -0.5``. ``algo``: "auto" takes
    for each document the kernel that is expected to be done sooner, reckoning with whole
    documents and full caches; "mma" and "tc" the mma.sync and the tcgen05 one for all.

    A handle is a plan for these lengths (made in 46 us for a few documents, 0.1 ms for 2000, 0.8 ms
    for 32000); keys in use that change from run to run are ``k_lens_ptr`` of :meth:`run`."""

    _destroy = "ah_attn_destroy"

    def __init__(self, q_offsets, k_offsets, q_heads: int, kv_heads: int, head_dim: int, scale: float | None = None,
                 cap: float = 0.0, mask: str = "full", prefix=None, slopes=None, dtype: str = "fp16",
                 algo: str = "auto", device: int = 0):
        super().__init__()
        qo, ko = _whole(q_offsets, "q_offsets"), _whole(k_offsets, "k_offsets")
        if qo.size < 1 or qo.size != ko.size:
            raise EngineHarnessError("q_offsets and k_offsets have one entry more than there are documents")
        docs = qo.size - 1
        pre = None if prefix is None else _whole(prefix, "prefix")
        if pre is not None and pre.size != docs:
            raise EngineHarnessError("prefix has one entry for each document")
        axes = 0
        if slopes is not None:
            slopes = np.asarray(slopes, dtype=np.float32)
            axes = slopes.shape[1] if slopes.ndim == 2 else -1
            slopes = _floats(slopes, (q_heads, axes), "slopes")
        d = _AttnDesc(_code(_DTYPES, dtype, "dtype"), q_heads, kv_heads, head_dim,
                      max(head_dim, 1) ** -0.5 if scale is None else scale, cap, _code(_MASKS, mask, "mask"), axes,
                      _code(_ALGOS, algo, "algo"))
        err = _err()
        self._check(self._lib.ah_attn_create(device, ctypes.byref(d), docs, qo.ctypes.data, ko.ctypes.data, _data(pre),
                                             _data(slopes), ctypes.byref(self._h), err, _ERR_LEN), err,
                    "attention create")
        self.docs, self.q_heads, self.kv_heads, self.head_dim = docs, q_heads, kv_heads, head_dim

    def run(self, q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, q_pos_ptr: int = 0, k_pos_ptr: int = 0,
            k_lens_ptr: int = 0, q_strides=(0, 0), k_strides=(0, 0), v_strides=(0, 0), out_strides=(0, 0),
            stream: int = 0):
        """Strides are (token, head). ``q_pos_ptr`` / ``k_pos_ptr``: fp32 [axes][tokens].
        ``k_lens_ptr``: int32 [documents] on the device, the keys in use of each document."""
        io = _AttnIo(q_ptr, k_ptr, v_ptr, out_ptr, *q_strides, *k_strides, *v_strides, *out_strides, q_pos_ptr,
                     k_pos_ptr, k_lens_ptr)
        err = _err()
        self._check(self._lib.ah_attn_run(self._h, ctypes.byref(io), stream or None, err, _ERR_LEN), err,
                    "attention run")

    def status(self) -> int:
        """The device error word (0 = none), read and cleared: a pipeline wait that ran out.
        Synchronises the device."""
        st = ctypes.c_uint32(0)
        if self._lib.ah_attn_status(self._h, ctypes.byref(st)) != 0:
            raise EngineHarnessError("attention status read failed")
        return st.value
