"""Operators for training and serving scorers, on CUDA tensors and the current stream.

* ``qk_norm_rope``: RMS norm of every query and key head with a learned gain, and the rotation by position.
* ``relative_attention``: softmax attention with a learned bias per head and distance bucket.
* ``distill_top_logits`` / ``distill_top_logits_step``: how far a student's logits are from a teacher's top entries.

All three run hand-written kernels of libmgbs_b200.so and take part in autograd (first derivatives, in reverse mode; forward
mode, tracing and torch.func transforms are refused, and torch.compile wants the call inside torch.compiler.disable).
Wrong shapes, types or devices raise RuntimeError before anything is enqueued; there is no CPU fallback.  Nothing is kept
between calls, outputs and workspaces come from torch's allocator, equal calls give equal bits, and every call may be
captured in a CUDA graph (a backward pass only while no eager autograd graph of the same leaves is alive, a rule of
autograd's own).  TransformerValueScorer, TransformerValueNet and MLPActionScorer.distillation_loss call them.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_P, _I32, _I64 = C.c_void_p, C.c_int32, C.c_int64
_S3 = _I64 * 3
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # MGBS_DT_*
MAX_ENTRIES = 1024  # MGBS_DISTILL_MAX_ENTRIES


class MgbsQkNormArgs(C.Structure):
    _fields_ = [
        ("dtype", _I32), ("head_dim", _I32), ("heads_q", _I32), ("heads_k", _I32), ("interleaved", _I32),
        ("position_bits", _I32), ("batch", _I64), ("tokens", _I64),
        ("q_stride", _S3), ("k_stride", _S3), ("q_out_stride", _S3), ("k_out_stride", _S3), ("dq_out_stride", _S3),
        ("dk_out_stride", _S3), ("position_stride", _I64 * 2),
        ("q", _P), ("k", _P), ("q_out", _P), ("k_out", _P), ("q_gain", _P), ("k_gain", _P), ("phase", _P),
        ("positions", _P), ("dq_out", _P), ("dk_out", _P), ("dq_gain", _P), ("dk_gain", _P), ("workspace", _P),
        ("eps", C.c_float), ("reserved", _I32),
    ]


class MgbsRelAttentionArgs(C.Structure):
    _fields_ = [
        ("dtype", _I32), ("head_dim", _I32), ("heads", _I32), ("heads_kv", _I32), ("batch", _I64), ("tokens", _I64),
        ("q_stride", _S3), ("k_stride", _S3), ("v_stride", _S3), ("dout_stride", _S3),
        ("q", _P), ("k", _P), ("v", _P), ("table", _P), ("bucket_map", _P), ("bucket_order", _P), ("bucket_start", _P),
        ("lengths", _P), ("out", _P), ("stats", _P),
        ("num_buckets", _I32), ("max_distance", _I32), ("causal", _I32), ("scale", C.c_float),
        ("dout", _P), ("dq", _P), ("dk", _P), ("dv", _P), ("dtable", _P), ("workspace", _P), ("error", _P),
    ]


class MgbsDistillArgs(C.Structure):
    _fields_ = [
        ("dtype", _I32), ("entries", _I32), ("rows", _I64), ("width", _I32), ("index_bits", _I32),
        ("row_stride", _I64), ("grad_stride", _I64), ("teacher_stride", _I64), ("index_stride", _I64),
        ("logits", _P), ("teacher", _P), ("index", _P), ("row_weight", _P), ("loss", _P), ("grad", _P),
        ("temperature", C.c_float), ("reserved", _I32),
    ]


_SIGS = {
    "mgbs_sizeof_qk_norm_args": (C.c_int, []),
    "mgbs_qk_norm_rope": (C.c_int, [C.POINTER(MgbsQkNormArgs), _P]),
    "mgbs_qk_norm_rope_backward_workspace": (_I64, [_I32]),
    "mgbs_qk_norm_rope_backward": (C.c_int, [C.POINTER(MgbsQkNormArgs), _P]),
    "mgbs_sizeof_rel_attention_args": (C.c_int, []),
    "mgbs_rel_attention": (C.c_int, [C.POINTER(MgbsRelAttentionArgs), _P]),
    "mgbs_rel_attention_backward_workspace": (_I64, [C.POINTER(MgbsRelAttentionArgs)]),
    "mgbs_rel_attention_backward": (C.c_int, [C.POINTER(MgbsRelAttentionArgs), _P]),
    "mgbs_sizeof_distill_args": (C.c_int, []),
    "mgbs_distill_top_logits": (C.c_int, [C.POINTER(MgbsDistillArgs), _P]),
}
_lib.SIGNATURES.update(_SIGS)

_ready = None


def _load():
    global _ready
    if _ready is None:
        lib = _lib.load()
        for name, (res, args) in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        for size, mirror in ((lib.mgbs_sizeof_qk_norm_args, MgbsQkNormArgs), (lib.mgbs_sizeof_rel_attention_args, MgbsRelAttentionArgs),
                             (lib.mgbs_sizeof_distill_args, MgbsDistillArgs)):
            if size() != C.sizeof(mirror):
                raise RuntimeError(f"structure layout mismatch between operators.py and libmgbs_b200.so ({mirror.__name__})")
        _ready = lib
    return _ready


def _current_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same handle without a Stream object around it, where torch has the call: two microseconds of a small call's ten
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


def _enqueue(fn, args, device: torch.device, what: str) -> None:
    """Run a C entry on the tensors' device and that device's current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(C.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(C.byref(args), _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _refuse(what: str, why: str):
    raise RuntimeError(f"{what}: {why}")


def _once(backward):
    """once_differentiable where a graph of the gradient is being built; without its five microseconds elsewhere."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def _refuse_unseen(what: str, *tensors) -> None:
    """Refuse the transforms that would not see the kernel, and go on without its work or its tangent."""
    if torch.jit.is_tracing() or (torch._C._len_torch_dispatch_stack() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        _refuse(what, "cannot be recorded by torch.jit.trace or make_fx")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _refuse(what, "has no forward-mode derivative")


def _same_device(what: str, device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            _refuse(what, f"tensors on {device} and {t.device}")


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Uninitialised memory like t, contiguous."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor with its last dimension dense (a copy only where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """Batch, token and head strides; a dimension of one entry has none."""
    s0, s1, s2, _ = t.stride()
    n0, n1, n2, _ = t.shape
    return (s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """A 16-bit tensor with rows on 16-byte boundaries (a copy only where they are not)."""
    t = _rows(t)
    s0, s1, s2 = _strides(t)
    if not (t.data_ptr() % 16 or (s0 | s1 | s2) % 8):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# ----------------------------------------------------------------------------------------------
# Query and key norm with the position rotation
# ----------------------------------------------------------------------------------------------


class RotaryFrequencies:
    """Rotation angles of the head_dim / 2 pairs of a head: position * base ** (-2 i / head_dim), or position *
    inv_freq[i].  Built once per model.  Held as 64-bit fractions of a turn, so that angles keep float32 accuracy at any
    64-bit position."""

    def __init__(self, head_dim: int, base: float = 10000.0, inv_freq: Optional[Sequence[float]] = None, device=None):
        if head_dim < 2 or head_dim % 2:
            raise RuntimeError("RotaryFrequencies: head_dim must be even")
        if inv_freq is None:
            if not base > 0.0 or math.isinf(base):
                raise RuntimeError("RotaryFrequencies: base must be positive and finite")
            inv_freq = [float(base) ** (-2.0 * i / head_dim) for i in range(head_dim // 2)]
        inv_freq = [float(f) for f in inv_freq]
        if len(inv_freq) != head_dim // 2 or not all(math.isfinite(f) for f in inv_freq):
            raise RuntimeError("RotaryFrequencies: inv_freq needs head_dim / 2 finite values")
        turns = [round(math.ldexp(f / (2.0 * math.pi) % 1.0, 64)) % (1 << 64) for f in inv_freq]
        self.head_dim, self.inv_freq = int(head_dim), inv_freq
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.phase = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=dev)


def _qk_args(q, k, q_gain, k_gain, rotary, positions, eps, interleaved) -> MgbsQkNormArgs:
    a = MgbsQkNormArgs()
    a.dtype, a.head_dim, a.heads_q, a.heads_k = DTYPES[q.dtype], q.shape[3], q.shape[2], k.shape[2]
    a.batch, a.tokens, a.interleaved, a.eps = q.shape[0], q.shape[1], int(interleaved), eps
    a.q_stride[:], a.k_stride[:] = _strides(q), _strides(k)
    a.q, a.k = q.data_ptr(), k.data_ptr()
    a.q_gain, a.k_gain, a.phase = q_gain.data_ptr(), k_gain.data_ptr(), rotary.phase.data_ptr()
    if positions is not None:
        a.position_bits, a.positions = positions.element_size() * 8, positions.data_ptr()
        a.position_stride[:] = (positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1))
    return a


def _qk_forward(q, k, q_gain, k_gain, rotary, positions, eps, interleaved):
    a = _qk_args(q, k, q_gain, k_gain, rotary, positions, eps, interleaved)
    q_out, k_out = _dense(q), _dense(k)
    a.q_out_stride[:], a.k_out_stride[:] = _strides(q_out), _strides(k_out)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    _enqueue(_load().mgbs_qk_norm_rope, a, q.device, "qk_norm_rope")
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_gain, k_gain, rotary, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_gain, k_gain, positions)
        ctx.rotary, ctx.eps, ctx.interleaved = rotary, eps, interleaved
        return _qk_forward(q, k, q_gain, k_gain, rotary, positions, eps, interleaved)

    @staticmethod
    @_once
    def backward(ctx, dq_out, dk_out):
        _refuse_unseen("qk_norm_rope backward", dq_out, dk_out)
        q, k, q_gain, k_gain, positions = ctx.saved_tensors
        lib = _load()
        a = _qk_args(q, k, q_gain, k_gain, ctx.rotary, positions, ctx.eps, ctx.interleaved)
        dq_out, dk_out = _rows(dq_out), _rows(dk_out)
        dq, dk, dq_gain, dk_gain = _dense(q), _dense(k), _dense(q_gain), _dense(k_gain)
        work = q_gain.new_empty(lib.mgbs_qk_norm_rope_backward_workspace(q.shape[3]) // 4)
        a.q_out_stride[:], a.k_out_stride[:] = _strides(dq), _strides(dk)
        a.dq_out_stride[:], a.dk_out_stride[:] = _strides(dq_out), _strides(dk_out)
        a.q_out, a.k_out, a.dq_out, a.dk_out = dq.data_ptr(), dk.data_ptr(), dq_out.data_ptr(), dk_out.data_ptr()
        a.dq_gain, a.dk_gain, a.workspace = dq_gain.data_ptr(), dk_gain.data_ptr(), work.data_ptr()
        _enqueue(lib.mgbs_qk_norm_rope_backward, a, q.device, "qk_norm_rope backward")
        return dq, dk, dq_gain, dk_gain, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_gain: torch.Tensor, k_gain: torch.Tensor, rotary: RotaryFrequencies,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, k) with every head normalised, scaled and rotated: R(position) (gain * x / sqrt(mean(x^2) + eps)).

    ``q`` [batch, tokens, heads, head_dim], ``k`` [batch, tokens, key heads, head_dim]: bfloat16, float16 or float32 (one
    type), any strides (a copy is made only if the last dimension is not dense), head_dim even up to 256.  Gains:
    float32 [head_dim].  ``positions``: int32 or int64 [tokens] or [batch, tokens], negative ones included; by default a
    token's index.  Pairs are (i, i + head_dim / 2), or (2 i, 2 i + 1) with ``interleaved``.  Statistics and rotation are
    in float32 (a head's sum of squares has to stay below 3e38), rounded once.  Differentiable in q, k and the gains."""
    what, dtype, device = "qk_norm_rope", q.dtype, q.device
    _refuse_unseen(what, q, k, q_gain, k_gain)
    if not q.is_cuda or q.dim() != 4 or k.dim() != 4:
        _refuse(what, "q and k must be [batch, tokens, heads, head_dim] CUDA tensors")
    if dtype not in DTYPES or k.dtype != dtype:
        _refuse(what, "q and k must have one type: bfloat16, float16 or float32")
    (b, t, h, d), (kb, kt, kh, kd) = q.shape, k.shape
    if (kb, kt, kd) != (b, t, d):
        _refuse(what, "q and k must agree in batch, tokens and head_dim")
    if not 2 <= d <= 256 or d % 2 or h < 1 or kh < 1:
        _refuse(what, "head_dim must be even, 2 to 256, with one head at least")
    if d != rotary.head_dim:
        _refuse(what, f"the frequencies are for head_dim {rotary.head_dim}")
    if q_gain.dtype != torch.float32 or k_gain.dtype != torch.float32 or q_gain.shape != (d,) or k_gain.shape != (d,):
        _refuse(what, "gains must be float32 [head_dim]")
    if not (eps >= 0.0 and math.isfinite(eps)):
        _refuse(what, "eps must not be negative")
    if positions is not None:
        if positions.dtype is not torch.int64 and positions.dtype is not torch.int32:
            _refuse(what, "positions must be int32 or int64")
        if positions.shape != (t,) and positions.shape != (b, t):
            _refuse(what, "positions must be [tokens] or [batch, tokens]")
    _same_device(what, device, k, q_gain, k_gain, positions, rotary.phase)
    q, k, q_gain, k_gain = _rows(q), _rows(k), q_gain.contiguous(), k_gain.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_gain.requires_grad or k_gain.requires_grad):
        return _QkNormRope.apply(q, k, q_gain, k_gain, rotary, positions, float(eps), bool(interleaved))
    return _qk_forward(q, k, q_gain, k_gain, rotary, positions, float(eps), bool(interleaved))


# ----------------------------------------------------------------------------------------------
# Attention with a learned relative bias
# ----------------------------------------------------------------------------------------------


def relative_bucket(offset: int, num_buckets: int, max_distance: int, causal: bool) -> int:
    """Bucket of a key `offset` places after its query (negative: before).  Keys after the query have the upper half of
    the buckets (none with ``causal``, where they share bucket 0).  Half of a side's buckets hold one distance each; the
    others cover [exact, max_distance) in equal factors and the last takes all from there on.  Borders are decided in
    whole numbers."""
    side = num_buckets if causal else num_buckets // 2
    n = max(-offset, 0) if causal else abs(offset)
    first = 0 if causal or offset <= 0 else side
    exact = side // 2
    if n < exact or side == 1:
        return first + min(n, side - 1)
    steps, grown = side - exact, 0
    if exact == 0:
        return first + side - 1
    # the largest s with n >= exact * (max_distance / exact) ** (s / steps)
    while grown < steps - 1 and n ** steps * exact ** (grown + 1) >= max_distance ** (grown + 1) * exact ** steps:
        grown += 1
    return first + exact + grown


class RelativeBuckets:
    """Which learned bias a pair of positions takes: ``num_buckets`` buckets of key minus query, exact for near
    distances and growing by equal factors up to ``max_distance`` (see relative_bucket).  ``causal`` also hides keys
    after their query.  Built once per model.  ``error_code()`` is 0 unless a kernel of a call with these buckets gave up
    waiting for its own copies or products, which leaves NaN in the rows concerned."""

    def __init__(self, num_buckets: int = 32, max_distance: int = 128, causal: bool = False, device=None):
        self.num_buckets, self.max_distance, self.causal = int(num_buckets), int(max_distance), bool(causal)
        least = 2 if causal else 4
        if not least <= self.num_buckets <= 512 or (not causal and self.num_buckets % 2):
            raise RuntimeError(f"RelativeBuckets: num_buckets must be {least} to 512" + ("" if causal else " and even"))
        if not (self.num_buckets if causal else self.num_buckets // 2) // 2 < self.max_distance <= 1024:
            raise RuntimeError("RelativeBuckets: max_distance must be over the one-distance buckets of a side and at most 1024")
        m = self.max_distance
        buckets = [relative_bucket(o, self.num_buckets, m, self.causal) for o in range(-m, m + 1)]
        order = sorted(range(2 * m + 1), key=lambda i: buckets[i])
        start = [0] * (self.num_buckets + 1)
        for b in buckets:
            start[b + 1] += 1
        for b in range(self.num_buckets):
            start[b + 1] += start[b]
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        packed = torch.tensor(buckets + order + start + [0], dtype=torch.int32, device=dev)
        n = 2 * m + 1
        self.map, self.order, self.start = packed[:n], packed[n:2 * n], packed[2 * n:-1]
        self.error = packed[-1:]

    def error_code(self) -> int:
        """Waits for the calls before it."""
        return int(self.error.item())


def _rel_args(q, k, v, table, buckets, lengths, scale) -> MgbsRelAttentionArgs:
    a = MgbsRelAttentionArgs()
    a.dtype, a.head_dim, a.heads, a.heads_kv = DTYPES[q.dtype], q.shape[3], q.shape[2], k.shape[2]
    a.batch, a.tokens, a.scale = q.shape[0], q.shape[1], scale
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    a.q, a.k, a.v, a.table = q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr()
    a.bucket_map, a.bucket_order, a.bucket_start = buckets.map.data_ptr(), buckets.order.data_ptr(), buckets.start.data_ptr()
    a.error = buckets.error.data_ptr()
    a.num_buckets, a.max_distance, a.causal = buckets.num_buckets, buckets.max_distance, int(buckets.causal)
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    return a


def _rel_forward(q, k, v, table, buckets, lengths, scale, with_stats):
    a = _rel_args(q, k, v, table, buckets, lengths, scale)
    out = _dense(q)
    a.out = out.data_ptr()
    stats = None
    if with_stats:
        stats = torch.empty((q.shape[0], q.shape[2], q.shape[1], 2), dtype=torch.float32, device=q.device)
        a.stats = stats.data_ptr()
    _enqueue(_load().mgbs_rel_attention, a, q.device, "relative_attention")
    return out, stats


class _RelativeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, lengths, scale):
        # the backward of short sequences with a key head per query head makes its statistics anew
        out, stats = _rel_forward(q, k, v, table, buckets, lengths, scale, q.shape[1] > 64 or q.shape[2] != k.shape[2])
        ctx.save_for_backward(q, k, v, table, lengths, out, stats)
        ctx.buckets, ctx.scale = buckets, scale
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        _refuse_unseen("relative_attention backward", dout)
        q, k, v, table, lengths, out, stats = ctx.saved_tensors
        lib = _load()
        a = _rel_args(q, k, v, table, ctx.buckets, lengths, ctx.scale)
        dout = _aligned(dout)
        dq, dk, dv, dtable = _dense(q), _dense(k), _dense(v), _dense(table)
        work = table.new_empty(max(16, lib.mgbs_rel_attention_backward_workspace(C.byref(a))) // 2)  # 16-bit elements
        a.dout_stride[:] = _strides(dout)
        a.out, a.dout = out.data_ptr(), dout.data_ptr()
        if stats is not None:
            a.stats = stats.data_ptr()
        a.dq, a.dk, a.dv, a.dtable, a.workspace = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dtable.data_ptr(), work.data_ptr()
        _enqueue(lib.mgbs_rel_attention_backward, a, q.device, "relative_attention backward")
        return dq, dk, dv, dtable, None, None, None


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, buckets: RelativeBuckets,
                       lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax_j(scale q_i . k_j + table[bucket(j - i), head]) v_j for every query head; [batch, tokens, heads, head_dim].

    ``q`` [batch, tokens, heads, head_dim], ``k`` and ``v`` [batch, tokens, key heads, head_dim], ``table`` [num_buckets,
    heads]: bfloat16 or float16 (one type), head_dim 32 or 64, heads a multiple of the key heads.  Any strides (a copy
    is made only where rows do not lie on 16-byte boundaries).  ``lengths`` (int32 [batch]): tokens of a sequence from
    its length on are padding: what they hold has no influence (nothing may write there during the call all the same, as
    tiles are loaded whole), their outputs and gradients are 0.  ``scale``: head_dim ** -0.5 by default.  A row whose
    biases leave no key (all -inf) gives 0; finite biases beyond 1e38 * min(1, scale) in size are masks alike.  A NaN or
    an infinity in the values of a key that only a causal mask or a bias hides may reach rows beside it, as 0 times it.
    Sums over the keys are in float32 before a row is divided by its weights' total: values up to 1e28 are safe.
    Differentiable in q, k, v and table; P and the scores' gradients P (dP - delta) are rounded to the inputs' type on the
    way, so with float16 a loss scale has to keep the latter within the type's range, 6e-8 to 65504."""
    what, dtype, device = "relative_attention", q.dtype, q.device
    _refuse_unseen(what, q, k, v, table)
    if not q.is_cuda or q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        _refuse(what, "q, k and v must be [batch, tokens, heads, head_dim] CUDA tensors")
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype != dtype or v.dtype != dtype or table.dtype != dtype:
        _refuse(what, "q, k, v and table must have one type: bfloat16 or float16")
    (b, t, h, d), (kb, kt, kh, kd) = q.shape, k.shape
    if (kb, kt, kd) != (b, t, d) or v.shape != k.shape:
        _refuse(what, "q, k and v must agree in batch, tokens and head_dim")
    if d != 32 and d != 64:
        _refuse(what, "head_dim must be 32 or 64")
    if kh < 1 or not 1 <= h <= 1024 or h % kh:
        _refuse(what, "query heads (at most 1024) must be a multiple of the key heads")
    if t > 1 << 20:
        _refuse(what, "at most 2^20 tokens")
    if table.shape != (buckets.num_buckets, h):
        _refuse(what, "table must be [num_buckets, heads]")
    if lengths is not None:
        if lengths.shape != (b,) or lengths.dtype != torch.int32:
            _refuse(what, "lengths must be int32 [batch]")
        lengths = lengths.contiguous()
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        _refuse(what, "scale must be positive and finite")
    _same_device(what, device, k, v, table, buckets.map, lengths)
    q, k, v, table = _aligned(q), _aligned(k), _aligned(v), table.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad):
        return _RelativeAttention.apply(q, k, v, table, buckets, lengths, scale)
    return _rel_forward(q, k, v, table, buckets, lengths, scale, False)[0]


# ----------------------------------------------------------------------------------------------
# Distillation from a teacher's top entries
# ----------------------------------------------------------------------------------------------


def _distill_check(what, logits, teacher, index, temperature):
    _refuse_unseen(what, logits)
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in DTYPES or logits.shape[1] < 1:
        _refuse(what, "logits must be a [rows, width] CUDA tensor with one column at least: bfloat16, float16 or float32")
    if teacher.dim() != 2 or teacher.shape != index.shape or teacher.shape[0] != logits.shape[0]:
        _refuse(what, "teacher and index must be [rows, entries]")
    if not 1 <= teacher.shape[1] <= MAX_ENTRIES:
        _refuse(what, f"1 to {MAX_ENTRIES} entries per row")
    if teacher.dtype not in DTYPES:
        _refuse(what, "teacher must be bfloat16, float16 or float32")
    if index.dtype is not torch.int64 and index.dtype is not torch.int32:
        _refuse(what, "index must be int32 or int64")
    if not 1e-30 <= temperature <= 1e30:
        _refuse(what, "temperature must be positive and finite")
    _same_device(what, logits.device, teacher, index)


def _float(teacher: torch.Tensor) -> torch.Tensor:
    teacher = teacher.detach()
    return teacher if teacher.dtype is torch.float32 else teacher.float()


def _distill_run(what, logits, teacher, index, temperature, weight, with_grad):
    a = MgbsDistillArgs()
    (rows, width), entries = logits.shape, teacher.shape[1]
    loss = teacher.new_empty(rows)
    grad = _dense(logits) if with_grad else None
    a.dtype, a.entries, a.rows, a.width = DTYPES[logits.dtype], entries, rows, width
    a.index_bits, a.temperature = index.element_size() * 8, temperature
    a.row_stride, a.teacher_stride, a.index_stride = logits.stride(0), teacher.stride(0), index.stride(0)
    a.logits, a.teacher, a.index, a.loss = logits.data_ptr(), teacher.data_ptr(), index.data_ptr(), loss.data_ptr()
    if with_grad:
        a.grad, a.grad_stride = grad.data_ptr(), grad.stride(0)
        if weight is not None:
            a.row_weight = weight.data_ptr()
    _enqueue(_load().mgbs_distill_top_logits, a, logits.device, what)
    return loss, grad


class _DistillTopLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, temperature):
        ctx.save_for_backward(logits, teacher, index)
        ctx.temperature = temperature
        return _distill_run("distill_top_logits", logits, teacher, index, temperature, None, False)[0]

    @staticmethod
    @_once
    def backward(ctx, dloss):
        _refuse_unseen("distill_top_logits backward", dloss)
        logits, teacher, index = ctx.saved_tensors
        weight = dloss.to(torch.float32).contiguous()
        return _distill_run("distill_top_logits backward", logits, teacher, index, ctx.temperature, weight, True)[1], None, None, None


def distill_top_logits(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                       temperature: float = 1.0) -> torch.Tensor:
    """Divergence of a student from a teacher's top entries, per row (float32 [rows]):
    sum_k p_k (log p_k - log softmax(logits / temperature)[index_k]) with p = softmax(teacher_logits / temperature).

    ``logits`` [rows, width]: bfloat16, float16 or float32.  ``teacher_logits`` and ``teacher_index`` (int32 or int64)
    [rows, entries], 1 to 1024 entries in any order; entries whose index lies outside [0, width) are padding, an index
    given twice counts with both probabilities, and a row without entries has loss 0.  Differentiable in logits (the
    teacher is a constant); a training loop that wants loss and gradient from one read of the logits calls
    distill_top_logits_step."""
    temperature = float(temperature)
    _distill_check("distill_top_logits", logits, teacher_logits, teacher_index, temperature)
    logits, teacher, index = _rows(logits), _rows(_float(teacher_logits)), _rows(teacher_index)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillTopLogits.apply(logits, teacher, index, temperature)
    return _distill_run("distill_top_logits", logits, teacher, index, temperature, None, False)[0]


def distill_top_logits_step(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, temperature: float = 1.0,
                            row_weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [rows], gradient [rows, width] of sum(row_weight * loss)) of distill_top_logits in one pass, outside autograd:
    ``logits.backward(gradient)`` carries it on.  ``row_weight``: float32 [rows], 1 by default."""
    what = "distill_top_logits_step"
    temperature = float(temperature)
    _distill_check(what, logits, teacher_logits, teacher_index, temperature)
    if row_weight is not None:
        if row_weight.dtype != torch.float32 or row_weight.shape != logits.shape[:1]:
            _refuse(what, "row_weight must be float32 [rows]")
        _same_device(what, logits.device, row_weight)
        row_weight = row_weight.detach().contiguous()
    return _distill_run(what, _rows(logits.detach()), _rows(_float(teacher_logits)), _rows(teacher_index), temperature, row_weight, True)
