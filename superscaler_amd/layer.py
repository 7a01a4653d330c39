"""The operators of a transformer layer's training step that are no plain matrix products, on libace_layer.so (include/ace_layer.h).

What a profile database of a layer is taken of on an MI355X (superscaler_amd.profile_layer does that), and the optimizer step
whose state bytes the memory model counts:

  block_norm, block_norm_backward               norm at a block's exit, gate, scaled residual, norm at the next block's entry
  window_attention, window_attention_backward   causal attention over a window of keys and a few first ones; prompts and single tokens
  AdamW                                         one step over many tensors at once, moments in 32 or 8 bits

Tensors live on a GPU; work goes to the stream that is current on their device, and nothing waits for it.  A tensor last used on
another stream is the caller's to order.  Where a row's elements are not adjacent the call works on a contiguous copy.  Other shapes and
sizes raise ValueError, other types TypeError, a missing library or a HIP failure AceError.  There is no other form behind these calls.

Gradients come from the *_backward calls; torch's automatic differentiation records nothing of these operators.  Where it is on and an
input requires a gradient, so do the results, and going backward through them raises AceError: no gradient is lost unnoticed.
"""
import ctypes
import math
import os
import struct
from typing import NamedTuple, Optional

import numpy as np
import torch

from .evaluator import ACE_ETOOBIG, AceError

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libace_layer.so")
_lib = None

EXPORTS = ["ace_layer_abi_version", "ace_layer_strerror", "ace_layer_last_hip_error", "ace_block_norm_forward", "ace_block_norm_workspace_bytes",
           "ace_block_norm_backward", "ace_attend_workspace_bytes", "ace_attend_forward", "ace_attend_backward_workspace_bytes",
           "ace_attend_backward", "ace_adamw_step", "ace_adamw_moments"]
ABI_VERSION = 1
MAX_WIDTH = 32768       # ACE_NORM_MAX_WIDTH
MAX_HEAD = 128
ADAMW_BLOCK, ADAMW_CHUNK = 256, 8192

_NONE = 3
_LONGEST = (1 << 31) - 1
_HALVES = (torch.bfloat16, torch.float16)
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


# ace_block_norm_t: rows, rows_per_gate; width, dtype, layer; residual_scale, eps; seven pointers (packed: a third of the time that a
# ctypes structure takes, on a call that a single token waits for)
_BLOCK_NORM = struct.Struct("=2q3i2f4x7Q")
# ace_attend_t: batch, queries, keys, heads, kv_heads, dim, dtype, window, sinks; scale; start and length; four times three strides;
# q, k, v, out and lse
_ATTEND = struct.Struct("=9if2Q12q5Q")


class _AdamW(ctypes.Structure):
    _fields_ = [("d_tensors", _vp), ("d_chunk_tensor", _vp), ("n_tensors", _i32), ("n_chunks", _i64), ("state_bits", _i32), ("grad_type", _i32),
                ("copy_type", _i32), ("d_m", _vp), ("d_v", _vp), ("d_m_scale", _vp), ("d_v_scale", _vp)]


def load_library():
    """dlopen the in-tree HIP library; no fallback of any kind."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(_LIB_PATH):
        raise AceError(f"{_LIB_PATH} is missing: build it with `python -m superscaler_amd.build`")
    lib = ctypes.CDLL(_LIB_PATH)
    for name in EXPORTS:
        getattr(lib, name).restype = ctypes.c_int
    for name in ("ace_layer_strerror", "ace_layer_last_hip_error"):
        getattr(lib, name).restype = ctypes.c_char_p
    for name in ("ace_block_norm_workspace_bytes", "ace_attend_workspace_bytes", "ace_attend_backward_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    lib.ace_layer_strerror.argtypes = [ctypes.c_int]
    lib.ace_block_norm_forward.argtypes = [_vp] * 5
    lib.ace_block_norm_workspace_bytes.argtypes = [_vp]
    lib.ace_block_norm_backward.argtypes = [_vp] * 12 + [ctypes.c_size_t, _vp]
    lib.ace_attend_workspace_bytes.argtypes = [_vp]
    lib.ace_attend_forward.argtypes = [_vp, _vp, ctypes.c_size_t, _vp]
    lib.ace_attend_backward_workspace_bytes.argtypes = [_vp]
    lib.ace_attend_backward.argtypes = [_vp] * 7 + [ctypes.c_size_t, _vp]
    lib.ace_adamw_step.argtypes = [_vp] * 4 + [_f32] * 8 + [_vp]
    lib.ace_adamw_moments.argtypes = [_vp] * 4 + [_i64, _vp, _vp, _vp]
    if lib.ace_layer_abi_version() != ABI_VERSION:
        raise AceError("libace_layer.so has a different ABI version")
    _lib = lib
    return lib


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, name, *args):
    """A call of the library on `device` and its current stream."""
    lib, index = _lib or load_library(), device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            rc = getattr(lib, name)(*args, _raw_stream(index))
    else:
        rc = getattr(lib, name)(*args, _raw_stream(index))
    if rc != 0:
        if rc == ACE_ETOOBIG:
            raise ValueError(f"{name}: {lib.ace_layer_strerror(rc).decode()}")
        hip = lib.ace_layer_last_hip_error().decode() if rc == -3 else ""
        raise AceError(f"{name}: {lib.ace_layer_strerror(rc).decode()}" + (f" ({hip})" if hip else ""))


def _pointer(t):
    return None if t is None else t.data_ptr()


def _on_gpu(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: a tensor expected, not {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{what} is not on a GPU: these operators run on the HIP kernels only")


class _Untracked(torch.autograd.Function):
    """Results that automatic differentiation cannot go through: the first `n` of the tensors, which depend on the others."""
    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise AceError(f"{ctx.name} is not recorded by automatic differentiation: its gradients come from {ctx.name}_backward (call it under torch.no_grad())")


def _lost(*inputs):
    """Whether automatic differentiation would miss a gradient of these."""
    for t in inputs:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


def _untracked(name, results, inputs):
    made = iter(_Untracked.apply(name, sum(t is not None for t in results), *(t for t in results + inputs if t is not None)))
    return [None if t is None else next(made) for t in results]


# ---- norms around a block ---------------------------------------------------------------------------------------------------
class BlockNorm(NamedTuple):
    """`residual`: the new residual stream (`x` itself where no block was given), `normed`: what the next block reads (None
    without an entry norm), `stats`: float32 [rows, 4], for block_norm_backward."""
    residual: torch.Tensor
    normed: Optional[torch.Tensor]
    stats: torch.Tensor


class BlockNormGrads(NamedTuple):
    """Gradients of block_norm's arguments, None for those that were not given."""
    x: torch.Tensor
    block: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    exit_weight: Optional[torch.Tensor]
    exit_bias: Optional[torch.Tensor]
    entry_weight: Optional[torch.Tensor]
    entry_bias: Optional[torch.Tensor]


def _rows_per_gate(gate_shape, shape):
    """How many consecutive rows share a row of the gate, or None."""
    for k in range(len(shape) - 1, -1, -1):
        if gate_shape in (shape[:k] + shape[-1:], shape[:k] + (1,) * (len(shape) - 1 - k) + shape[-1:]):
            return max(1, math.prod(shape[k:-1]))
    return None


def _fits(t, dtype, device, shape):
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and (shape is None or t.shape == shape)


def _refuse_block_norm(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind):
    """Says what is wrong with arguments that do not fit together."""
    _on_gpu(x, "x")
    if x.dtype not in _TYPES:
        raise TypeError(f"x: float32, bfloat16 or float16 expected, not {x.dtype}")
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind: 'layer' or 'rms' expected, not {kind!r}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x: rows of 1 to {MAX_WIDTH} elements expected, got shape {tuple(x.shape)}")
    width = tuple(x.shape[-1:])
    for name, t, size in (("block", block, tuple(x.shape)), ("gate", gate, None), ("exit_weight", exit_weight, width), ("exit_bias", exit_bias, width),
                          ("entry_weight", entry_weight, width), ("entry_bias", entry_bias, width)):
        if t is None:
            continue
        _on_gpu(t, name)
        if t.dtype != x.dtype:
            raise TypeError(f"{name}: {x.dtype} expected like x, not {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
        if size is not None and tuple(t.shape) != size:
            raise ValueError(f"{name}: shape {size} expected, got {tuple(t.shape)}")
    if block is None and (gate is not None or exit_weight is not None or residual_scale != 1.0):
        raise ValueError("a gate, an exit norm and a residual scale go with a block")
    if (exit_bias is not None and exit_weight is None) or (entry_bias is not None and entry_weight is None):
        raise ValueError("a bias goes with its norm's weight")
    raise ValueError("neither a block nor an entry norm: nothing to compute")


def _block_norm_args(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind, eps):
    """(packed arguments, the tensors whose addresses they hold, rows)"""
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _TYPES and x.dim() > 0 and 1 <= x.shape[-1] <= MAX_WIDTH and kind in ("layer", "rms")):
        _refuse_block_norm(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind)
    dtype, device, shape = x.dtype, x.device, x.shape
    width = shape[-1:]
    if not ((block is None or _fits(block, dtype, device, shape)) and (gate is None or _fits(gate, dtype, device, None)) and
            (exit_weight is None or _fits(exit_weight, dtype, device, width)) and (exit_bias is None or _fits(exit_bias, dtype, device, width)) and
            (entry_weight is None or _fits(entry_weight, dtype, device, width)) and (entry_bias is None or _fits(entry_bias, dtype, device, width))) or \
            (exit_bias is not None and exit_weight is None) or (entry_bias is not None and entry_weight is None) or \
            (block is None and (entry_weight is None or gate is not None or exit_weight is not None or residual_scale != 1.0)):
        _refuse_block_norm(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind)
    per_gate = 1
    if gate is not None:
        per_gate = _rows_per_gate(tuple(gate.shape), tuple(shape))
        if per_gate is None:
            raise ValueError(f"gate: one row for all of x, or for each of its leading indices, expected; got {tuple(gate.shape)} for x {tuple(shape)}")
    keep = [t if t is None else t.contiguous() for t in (x, block, gate, exit_weight, exit_bias, entry_weight, entry_bias)]
    rows = x.numel() // width[0]
    a = _BLOCK_NORM.pack(rows, per_gate, width[0], _TYPES[dtype], kind == "layer", residual_scale, eps, *[0 if t is None else t.data_ptr() for t in keep])
    return a, keep, rows


def block_norm(x, block=None, *, residual_scale=1.0, gate=None, exit_weight=None, exit_bias=None, entry_weight=None, entry_bias=None, kind="layer",
               eps=1e-5) -> BlockNorm:
    """The step between two blocks of a layer, row by row over the last dimension, in one pass:

        residual = residual_scale * x + gate * (N(block) * exit_weight + exit_bias)
        normed   = N(residual) * entry_weight + entry_bias

    N: (u - mean u) / sqrt(var u + eps) (`kind` "layer") or u / sqrt(mean u^2 + eps) ("rms").  Without exit_weight the block is
    taken as it is, without entry_weight there is no `normed`, without a block it is the entry norm of x alone.  `gate`: one row
    [width], or one for each of x's leading indices ([batch, width] for x [batch, length, width], or x's own shape).  All tensors are
    of one type; `normed` is computed from the residual before that is rounded to it."""
    a, keep, rows = _block_norm_args(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind, eps)
    x0 = keep[0]   # (contiguous: so is what is made like it)
    residual = x if block is None else torch.empty_like(x0)
    normed = None if entry_weight is None else torch.empty_like(x0)
    stats = x0.new_empty((rows, 4), dtype=torch.float32)
    _call(x0.device, "ace_block_norm_forward", a, None if block is None else residual.data_ptr(), _pointer(normed), stats.data_ptr())
    if _lost(x, block, gate, exit_weight, exit_bias, entry_weight, entry_bias):
        made = _untracked("block_norm", (None if block is None else residual, normed, stats), (x, block, gate, exit_weight, exit_bias, entry_weight, entry_bias))
        return BlockNorm(residual if block is None else made[0], *made[1:])
    return BlockNorm(residual, normed, stats)


def block_norm_backward(d_residual, d_normed, x, block, stats, *, residual_scale=1.0, gate=None, exit_weight=None, exit_bias=None, entry_weight=None,
                        entry_bias=None, kind="layer") -> BlockNormGrads:
    """Gradients of what block_norm was given, from those of its two results (either may be None) and its `stats`.  Sums over rows
    are in 32 bits and in an order that the sizes alone decide: the same call gives the same bits."""
    a, keep, rows = _block_norm_args(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind, 0.0)
    if d_normed is not None and entry_weight is None:
        raise ValueError("d_normed goes with an entry norm")
    grads = []
    for name, t in (("d_residual", d_residual), ("d_normed", d_normed)):
        if t is not None:
            _on_gpu(t, name)
            if t.dtype != x.dtype:
                raise TypeError(f"{name}: {x.dtype} expected like x, not {t.dtype}")
            if t.shape != x.shape or t.device != x.device:
                raise ValueError(f"{name}: {tuple(x.shape)} on {x.device} expected, got {tuple(t.shape)} on {t.device}")
            t = t.contiguous()
        grads.append(t)
    _on_gpu(stats, "stats")
    if stats.dtype != torch.float32 or tuple(stats.shape) != (rows, 4) or not stats.is_contiguous() or stats.device != x.device:
        raise ValueError(f"stats: what block_norm returned for {rows} rows expected")
    lib = load_library()
    out = [None if t is None else (torch.zeros if rows == 0 else torch.empty)(t.shape, dtype=t.dtype, device=t.device)
           for t in (x, block, gate, exit_weight, exit_bias, entry_weight, entry_bias)]
    workspace = torch.empty(lib.ace_block_norm_workspace_bytes(a), dtype=torch.uint8, device=x.device)
    _call(x.device, "ace_block_norm_backward", a, *map(_pointer, grads), stats.data_ptr(), *map(_pointer, out), workspace.data_ptr(),
          workspace.numel())
    return BlockNormGrads(*out)


# ---- attention over a window and a few first keys ----------------------------------------------------------------------------
def _heads(t, what, like=None):
    """A [batch, tokens, heads, size] tensor as the kernels read it, a head's elements adjacent and everything else at multiples of
    16 bytes, or a copy where it is not so; and its three strides."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 4 and (t.dtype in _HALVES if like is None else t.dtype is like.dtype and t.device == like.device)):
        _on_gpu(t, what)
        if t.dim() != 4:
            raise ValueError(f"{what}: [batch, tokens, heads, size] expected, got shape {tuple(t.shape)}")
        if t.dtype not in _HALVES or (like is not None and t.dtype != like.dtype):
            raise TypeError(f"{what}: {'bfloat16 or float16' if like is None else like.dtype} expected, not {t.dtype}")
        raise ValueError(f"{what} is on {t.device}, q on {like.device}")
    (batch, tokens, heads, size), (b, n, h, e) = t.shape, t.stride()
    b, n, h = b if batch > 1 else 0, n if tokens > 1 else 0, h if heads > 1 else 0
    if (size > 1 and e != 1) or (b | n | h) & 7 or n >= 1 << 23 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        b, n, h, _ = t.stride()
    return t, (b, n, h)


def _attend_args(q, k, v, window, sinks, scale, start, lengths):
    """(q, k and v as the kernels read them, the arguments' part before the strides, q's, k's and v's strides, (batch, heads, queries))"""
    q, q_strides = _heads(q, "q")
    (k, k_strides), (v, v_strides) = _heads(k, "k", q), _heads(v, "v", q)
    (batch, queries, heads, dim), (_, keys, kv_heads, _) = q.shape, k.shape
    if not 8 <= dim <= MAX_HEAD or dim % 8:
        raise ValueError(f"q: heads of a multiple of 8 elements up to {MAX_HEAD} expected, got {dim}")
    if k.shape != v.shape or k.shape[0] != batch or k.shape[3] != dim:
        raise ValueError(f"k and v: [{batch}, keys, heads, {dim}] expected, got {tuple(k.shape)} and {tuple(v.shape)}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads do not share {kv_heads} heads of keys evenly")
    if window is not None and window < 1 or sinks < 0:
        raise ValueError(f"window: None or at least 1, and sinks >= 0 expected, got {window} and {sinks}")
    scale = 1 / math.sqrt(dim) if scale is None else float(scale)
    if not 0 < scale <= 1e30:
        raise ValueError(f"scale: a positive number expected, got {scale}")
    for name, t in (("start", start), ("lengths", lengths)):
        if t is None:
            continue
        _on_gpu(t, name)
        if t.dtype != torch.int32:
            raise TypeError(f"{name}: int32 expected, not {t.dtype}")
        if tuple(t.shape) != (batch,) or t.device != q.device or not t.is_contiguous():
            raise ValueError(f"{name}: [{batch}] on {q.device} expected, got {tuple(t.shape)} on {t.device}")
    # (no key is outside of a window of 2^31 - 1)
    head = (batch, queries, keys, heads, kv_heads, dim, _TYPES[q.dtype], 0 if window is None else min(int(window), _LONGEST), min(int(sinks), _LONGEST), scale,
            0 if start is None else start.data_ptr(), 0 if lengths is None else lengths.data_ptr())
    return q, k, v, head, q_strides + k_strides + v_strides, (batch, heads, queries)


def window_attention(q, k, v, *, window=None, sinks=0, scale=None, start=None, lengths=None):
    """Causal attention whose queries see a window of keys and a few first ones: (out [batch, queries, heads, size] of q's type,
    lse float32 [batch, heads, queries]).

    q [batch, queries, heads, size], k and v [batch, keys, kv_heads, size], bfloat16 or float16, in any strides; consecutive
    heads // kv_heads heads share a head of keys.  Query i of sequence b stands at position p = start[b] + i and sees key j where
    j < lengths[b], j <= p and (p - j < window or j < sinks); `start` and `lengths` are int32 [batch], by default
    keys - queries and keys: new queries at the end of a full cache.  `window` None: all earlier keys.  `scale`: 1 / sqrt(size)
    by default.  A query that sees no key has out 0 and lse -inf.  Up to 2^28 queries and keys, and 2^22 of batch * heads * (blocks of 128
    queries + 1) and of batch * kv_heads * (blocks of 128 keys + 1).  What a query does not see, a number or not, does not reach it, nor
    the gradients of a key one that does not see it (a call that finds what is not finite in its answers looks again and
    takes up to fifteen times as long)."""
    q, k, v, head, strides, rows = _attend_args(q, k, v, window, sinks, scale, start, lengths)
    out = q.new_empty(q.shape)
    lse = q.new_empty(rows, dtype=torch.float32)
    a = _ATTEND.pack(*head, *strides, *out.stride()[:3], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr())
    size = load_library().ace_attend_workspace_bytes(a)
    workspace = q.new_empty(size, dtype=torch.uint8) if size else None
    _call(q.device, "ace_attend_forward", a, _pointer(workspace), size)
    if _lost(q, k, v):
        out, lse = _untracked("window_attention", (out, lse), (q, k, v))
    return out, lse


def window_attention_backward(d_out, q, k, v, out, lse, *, window=None, sinks=0, scale=None, start=None, lengths=None):
    """Gradients (dq, dk, dv) of window_attention's q, k and v from that of its `out`; `out` and `lse` are what it returned.  The
    same call gives the same bits."""
    q, k, v, head, strides, rows = _attend_args(q, k, v, window, sinks, scale, start, lengths)
    (d_out, d_strides), (out, out_strides) = _heads(d_out, "d_out", q), _heads(out, "out", q)
    if d_out.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"d_out and out: {tuple(q.shape)} expected, got {tuple(d_out.shape)} and {tuple(out.shape)}")
    _on_gpu(lse, "lse")
    if lse.dtype != torch.float32 or tuple(lse.shape) != rows or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse: what window_attention returned expected")
    a = _ATTEND.pack(*head, *strides, *out_strides, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr())
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    size = load_library().ace_attend_backward_workspace_bytes(a)
    workspace = q.new_empty(size, dtype=torch.uint8)
    _call(q.device, "ace_attend_backward", a, d_out.data_ptr(), (_i64 * 3)(*d_strides), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), workspace.data_ptr(), size)
    return dq, dk, dv


# ---- AdamW over many tensors ------------------------------------------------------------------------------------------------
class AdamW:
    """One step over many tensors at once:

        g = grad_scale * grad;  m = m b1 + g (1 - b1);  v = v b2 + g^2 (1 - b2)
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps);  copy = p rounded

    `params`: float32 tensors, updated in place; `copies`: None, or for each of them the bfloat16 or float16 tensor that the
    forward pass reads, written by every step.  `state_bits` 32: moments in float32 (8 bytes per weight).  8: in blocks of 256
    elements, m as int8 in steps of its largest magnitude / 127, sqrt(v) as uint8 in steps of its maximum / 255 (2 bytes per
    weight and 8 per block); a step computes with the new moments before they are rounded, and sqrt(v) is rounded to zero only
    where it is zero.  A block with a value that is not finite comes back as NaN.

    `state`: the moments, as flat tensors ("m", "v", and with 8 bits "m_scale", "v_scale"), to be saved and restored with copy_;
    tensor i's elements begin at `offsets[i]`, a multiple of 256.  The tensors' memory is taken down here: a step with a parameter or copy that
    has moved since raises ValueError, and needs a new AdamW."""

    def __init__(self, params, *, copies=None, state_bits=32):
        params = list(params)
        copies = [None] * len(params) if copies is None else list(copies)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits: 8 or 32 expected, not {state_bits!r}")
        if not params:
            raise ValueError("no parameters")
        if len(copies) != len(params):
            raise ValueError(f"{len(copies)} copies for {len(params)} parameters")
        self.copy_type = None if copies[0] is None else getattr(copies[0], "dtype", None)
        if self.copy_type not in (None, torch.bfloat16, torch.float16):
            raise TypeError(f"copies: bfloat16 or float16 expected, not {self.copy_type}")
        for i, (p, c) in enumerate(zip(params, copies)):
            _on_gpu(p, f"params[{i}]")
            if p.dtype != torch.float32:
                raise TypeError(f"params[{i}]: float32 expected, not {p.dtype}")
            if not p.is_contiguous() or p.device != params[0].device:
                raise ValueError(f"params[{i}]: a contiguous tensor on {params[0].device} expected")
            if (c is None) != (self.copy_type is None):
                raise ValueError("copies: for all parameters or for none")
            if c is not None:
                _on_gpu(c, f"copies[{i}]")
                if c.dtype != self.copy_type:
                    raise TypeError(f"copies[{i}]: {self.copy_type} expected, not {c.dtype}")
                if c.shape != p.shape or not c.is_contiguous() or c.device != p.device:
                    raise ValueError(f"copies[{i}]: a contiguous tensor like params[{i}] expected")
        load_library()
        self.params, self.copies, self.state_bits, self.device = params, copies, state_bits, params[0].device
        sizes = np.array([p.numel() for p in params], dtype=np.int64)
        padded, chunks = -(-sizes // ADAMW_BLOCK) * ADAMW_BLOCK, -(-sizes // ADAMW_CHUNK)
        self._first_chunks = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int64)
        ends = np.cumsum(padded)
        self.offsets, self.size = [int(e - p) for e, p in zip(ends, padded)], int(ends[-1])
        table = np.stack([np.array([p.data_ptr() for p in params], dtype=np.int64), np.array([0 if c is None else c.data_ptr() for c in copies], dtype=np.int64),
                          sizes, ends - padded, self._first_chunks[:-1]], axis=1)
        self._tensors = torch.from_numpy(np.ascontiguousarray(table)).to(self.device)
        self._chunk_tensor = torch.from_numpy(np.repeat(np.arange(len(params), dtype=np.int32), chunks)).to(self.device)
        code = torch.float32 if state_bits == 32 else None
        self.state = {"m": torch.zeros(self.size, dtype=code or torch.int8, device=self.device), "v": torch.zeros(self.size, dtype=code or torch.uint8, device=self.device)}
        if state_bits == 8:
            for name in ("m_scale", "v_scale"):
                self.state[name] = torch.zeros(self.size // ADAMW_BLOCK, dtype=torch.float32, device=self.device)
        self._shapes = [p.shape for p in params]
        self._places = table[:, 0].tolist(), table[:, 1].tolist()
        self._args = _AdamW(self._tensors.data_ptr(), self._chunk_tensor.data_ptr(), len(params), int(self._first_chunks[-1]), state_bits, 0,
                            _NONE if self.copy_type is None else _TYPES[self.copy_type])

    def _held(self):
        """The state's tensors, as they are now (a caller may have put others of the same kind in their place)."""
        for name, t in self.state.items():
            n = self.size // ADAMW_BLOCK if name.endswith("scale") else self.size
            kind = torch.float32 if self.state_bits == 32 or name.endswith("scale") else torch.int8 if name == "m" else torch.uint8
            if t.dtype != kind or t.dim() != 1 or t.shape[0] != n or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"state[{name!r}]: {n} contiguous elements of {kind} on {self.device} expected")
        return self.state["m"], self.state["v"], self.state.get("m_scale"), self.state.get("v_scale")

    def step(self, grads, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, step=1, grad_scale=None):
        """`grads`: a gradient for each parameter, all float32, bfloat16 or float16.  `step`: t, from 1.  `grad_scale`: None, or a
        float32 tensor of one element on the device that every gradient is multiplied with (a clipping factor)."""
        b1, b2 = betas
        if not (0 <= b1 < 1 and 0 <= b2 < 1) or step < 1 or eps < 0:
            raise ValueError(f"betas in [0, 1), a step from 1 and eps >= 0 expected, got {betas}, {step}, {eps}")
        grads = list(grads)
        if len(grads) != len(self._shapes):
            raise ValueError(f"{len(grads)} gradients for {len(self._shapes)} parameters")
        kind, device = getattr(grads[0], "dtype", None), self.device
        if kind not in _TYPES:
            raise TypeError(f"grads[0]: a float32, bfloat16 or float16 tensor expected, not {kind or type(grads[0]).__name__}")
        pointers = (_vp * len(grads))()
        for i, (g, shape) in enumerate(zip(grads, self._shapes)):
            if not isinstance(g, torch.Tensor) or g.dtype != kind:
                raise TypeError(f"grads[{i}]: {kind} expected like the first, not {getattr(g, 'dtype', type(g).__name__)}")
            if g.shape != shape or g.device != device or not g.is_contiguous():
                raise ValueError(f"grads[{i}]: a contiguous tensor {tuple(shape)} on {device} expected, got {tuple(g.shape)} on {g.device}")
            pointers[i] = g.data_ptr()
        for what, held, places in (("params", self.params, self._places[0]), ("copies", self.copies if self.copy_type else (), self._places[1])):
            for i, (t, at) in enumerate(zip(held, places)):
                if t.data_ptr() != at:
                    raise ValueError(f"{what}[{i}] has moved: its memory is not the one that this AdamW was made with")
        if grad_scale is not None:
            _on_gpu(grad_scale, "grad_scale")
            if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != device:
                raise ValueError(f"grad_scale: one float32 on {device} expected")
        a = self._args
        a.grad_type = _TYPES[kind]
        a.d_m, a.d_v, a.d_m_scale, a.d_v_scale = map(_pointer, self._held())
        _call(device, "ace_adamw_step", ctypes.byref(a), pointers, self._first_chunks.ctypes.data, _pointer(grad_scale), b1, 1 - b1, b2, 1 - b2,
              1 - lr * weight_decay, lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step), eps)
        torch.autograd.graph.increment_version(self.params if self.copy_type is None else self.params + self.copies)

    def moments(self):
        """(m, v) as flat float32 tensors, elements as in `offsets`: the state itself with 32 bits, with 8 bits new tensors of
        the values that the codes stand for."""
        m, v, m_scale, v_scale = self._held()
        if self.state_bits == 32:
            return m, v
        out = [torch.empty(self.size, dtype=torch.float32, device=self.device) for _ in range(2)]
        _call(self.device, "ace_adamw_moments", m.data_ptr(), v.data_ptr(), m_scale.data_ptr(), v_scale.data_ptr(), self.size // ADAMW_BLOCK,
              out[0].data_ptr(), out[1].data_ptr())
        return out[0], out[1]
