"""Device-resident work around the loss head in one training step (include/pcp_step.h):
rollout packing, gradient statistics, norm and clipping, and the Nesterov update, over torch tensors in HBM.

Mirrors RLShepherd.trainStep (src/nodes/controllers/rl_shepherd.zig:487-515 packing,
:600-641 statistics, :643-682 update loop) and the host optimizer
(src/optimizers/nesterov.zig); the arithmetic runs in libpcp_grpo.so.
"""
from __future__ import annotations

import array
import ctypes
import sys
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import (DType, FLAG_ASYNC, GradClipArgs, GradStats, NesterovManyArgs, NesterovMode, NormType, PcpError,
                   VerifyArgs, check, lib)
from .grpo import _TORCH_DTYPE, Context, _ptr, _stream_handle, call_scope, default_context, dtype_code


def pack_rollouts(prompt_tokens: torch.Tensor, prompt_offsets: torch.Tensor, completion_tokens: torch.Tensor,
                  completion_offsets: torch.Tensor, n_rows: int, seq_len: int, *, stream=None,
                  ctx: Context | None = None):
    """Pack ragged rollouts (prompt then completion, truncated at seq_len) into
    ids int64 [n_rows, seq_len] and mask f32 [n_rows, seq_len] on the device."""
    dev = prompt_offsets.device
    ctx = ctx or default_context(dev.index or 0)
    for t in (prompt_tokens, prompt_offsets, completion_tokens, completion_offsets):
        if t.dtype != torch.int64:
            raise PcpError(-2, "token arrays and offsets must be int64")
    R = prompt_offsets.numel() - 1
    if completion_offsets.numel() != R + 1:
        raise PcpError(-1, "prompt and completion offsets differ in length")
    ids = torch.empty((n_rows, seq_len), dtype=torch.int64, device=dev)
    mask = torch.empty((n_rows, seq_len), dtype=torch.float32, device=dev)
    pt = _ptr(prompt_tokens) if prompt_tokens.numel() else None
    ct = _ptr(completion_tokens) if completion_tokens.numel() else None
    check(lib().pcp_pack_rollouts(ctx.handle, pt, prompt_tokens.numel(), _ptr(prompt_offsets), ct,
                                  completion_tokens.numel(), _ptr(completion_offsets), R, n_rows, seq_len,
                                  _ptr(ids), _ptr(mask), _stream_handle(stream)), ctx.handle)
    return ids, mask


def grad_stats(grads, *, stream=None, ctx: Context | None = None) -> dict:
    """rl_shepherd.zig:600-641 over one f32 tensor or a list of them."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    ctx = ctx or default_context(grads[0].device.index or 0)
    st = GradStats()
    n = len(grads)
    counts = [g.numel() for g in grads]
    for g in grads:
        if g.dtype != torch.float32:
            raise PcpError(-2, "gradients must be f32")
    ptrs = (ctypes.c_void_p * n)(*[_ptr(g) if k else None for g, k in zip(grads, counts)])
    check(lib().pcp_grad_stats_compute_many(ctx.handle, n, ptrs, (ctypes.c_int64 * n)(*counts), 0, ctypes.byref(st),
                                            _stream_handle(stream)), ctx.handle)
    return {"sumsq": st.sumsq, "l2_norm": st.l2_norm, "max_abs": st.max_abs, "nan_count": st.nan_count,
            "inf_count": st.inf_count, "elements": st.elements}


@dataclass
class GradNorm:
    norm: torch.Tensor        # f32 scalar
    coef: torch.Tensor        # f32 scalar: what brings the gradients down to max_norm, at most 1


def _described(tensors, what: str, dtype: DType | None = None):
    """What ``_lib.describe`` says of a list, its tensors contiguous and, with dtype, of that type (or None)."""
    d = _lib.describe(tensors)
    if 0 in d[3]:
        raise PcpError(-1, f"{what} must be contiguous")
    if dtype is not None and d[2] != _code(dtype) * len(tensors):
        if any(t is not None and int(_TORCH_DTYPE.get(t.dtype, -1)) != dtype for t in tensors):
            raise PcpError(-2, f"{what} must be {dtype.name}")
    return d


def _code(dtype: DType) -> bytes:
    return int(dtype).to_bytes(4, sys.byteorder)


def _same_sizes(grads, *others) -> None:
    """The descriptions (name, description, tensors) hold the gradients' numbers of elements (or None)."""
    for name, d, ts in others:
        if d is not None and d[1] != grads[1]:
            counts = memoryview(grads[1]).cast("q")
            if len(ts) != len(counts) or any(t is not None and t.numel() != c for t, c in zip(ts, counts)):
                raise PcpError(-12, f"{name} must hold as many tensors as the gradients, of the same sizes")


def _one_device(*descriptions) -> int:
    found = {d[4] for d in descriptions if d is not None and d[4] != -3}
    return -3 if not found else found.pop() if len(found) == 1 else -2


def grad_norm(grads, max_norm: float = float("inf"), *, norm_type: int | str = NormType.l2,
              outputs: GradNorm | None = None, sync: bool = True, stream=None, ctx: Context | None = None) -> GradNorm:
    """The norm of all gradients together (a tensor or a list of them, f32, bf16 and f16 mixed) and the coefficient
    that brings it down to max_norm (rounded to f32), both left on the device (pcp_grad_clip without outputs): norm_type "l2"
    or "max".
    ``Nesterov.update_many`` and ``nesterov_update_many`` take the coefficient there. A norm that is not finite is
    reported, and its coefficient is NaN. sync=False only enqueues. An empty list's results are on the
    ctx's device, or device 0."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    return _grad_clip(grads, max_norm, norm_type, None, outputs, sync, stream, ctx)


def clip_grads(grads, max_norm: float, *, norm_type: int | str = NormType.l2, out=None, outputs: GradNorm | None = None,
               sync: bool = True, stream=None, ctx: Context | None = None) -> GradNorm:
    """``grad_norm``, and the gradients times its coefficient: in place, or into `out` (as many tensors of the same
    sizes, of any of the three types, such as the pieces of the flat f32 buffer that ``Nesterov.update_flat`` takes).
    Gradients whose norm is not finite are left (or copied) as they are."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    out = grads if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    return _grad_clip(grads, max_norm, norm_type, out, outputs, sync, stream, ctx)


def _grad_clip(grads, max_norm, norm_type, out, outputs, sync, stream, ctx) -> GradNorm:
    if isinstance(norm_type, str):
        try:
            norm_type = NormType[norm_type]
        except KeyError:
            raise PcpError(-1, f"unknown norm_type {norm_type!r}") from None
    g = _described(grads, "gradients")
    o = None if out is None else g if out is grads else _described(out, "out")
    _same_sizes(g, ("out", o, out))
    given = [] if outputs is None else [outputs.norm, outputs.coef]
    e = _described(given, "outputs", DType.f32)
    device = _one_device(g, o, e)
    ctx = ctx or default_context(max(device, 0))
    a = GradClipArgs()
    with call_scope.of_described(ctx, stream, device, grads, () if out is None or out is grads else out, given) as handle:
        if outputs is None:
            both = torch.empty(2, dtype=torch.float32, device=torch.device("cuda", ctx.device))
            outputs = GradNorm(both[0], both[1])
            a.norm, a.coef = both.data_ptr(), both.data_ptr() + 4
        else:
            if e[1] != _ONE + _ONE:
                raise PcpError(-1, "outputs do not fit the call: norm and coef f32 scalars")
            a.norm, a.coef = memoryview(e[0]).cast("q")
        a.n_tensors, a.grads, a.counts, a.dtypes = len(grads), g[0], g[1], g[2]
        if o is not None:
            a.out, a.out_dtypes = o[0], o[2]
        a.norm_type, a.max_norm = int(norm_type), max_norm
        a.flags = 0 if sync else FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_grad_clip(ctx.handle, ctypes.byref(a)), ctx.handle)
    return outputs


_ONE = (1).to_bytes(8, sys.byteorder)


def nesterov_update_many(params, velocities, grads, param_copies=None, *, coef: torch.Tensor | None = None,
                         learning_rate: float = 0.01, momentum: float = 0.9, mode: int | str = NesterovMode.sutskever,
                         sync: bool = True, stream=None, ctx: Context | None = None) -> None:
    """The Nesterov update of a list of parameters (f32) with their velocities (f32) and gradients (f32, bf16 or f16),
    each where it lies (pcp_nesterov_update_many): the gradients times coef (a device scalar, ``grad_norm``'s; a
    coefficient that is not finite skips the update), the updated weights also as bf16 into param_copies (a list of
    tensors, None among them where there is no copy).
    sync=False only enqueues."""
    params, velocities, grads = list(params), list(velocities), list(grads)
    copies = None if param_copies is None else list(param_copies)
    if not params and not grads and not velocities:
        return
    v = _described(velocities, "velocities", DType.f32)
    _update_many(ctx, params, v, velocities, grads, copies, coef, learning_rate, momentum, mode, sync, stream)


def _update_many(ctx, params, v, velocities, grads, copies, coef, learning_rate, momentum, mode, sync, stream):
    """v: the velocities' description, or the addresses of an optimizer's own (velocities is None then)."""
    if isinstance(mode, str):
        try:
            mode = NesterovMode[mode]
        except KeyError:
            raise PcpError(-1, f"unknown mode {mode!r}") from None
    g, p = _described(grads, "gradients"), _described(params, "parameters", DType.f32)
    c = None if copies is None else _described(copies, "param_copies", DType.bf16)
    _same_sizes(g, ("params", p, params), ("velocities", None if velocities is None else v, velocities),
                ("param_copies", c, copies))
    scale = [] if coef is None else [coef]
    e = _described(scale, "coef", DType.f32)
    if coef is not None and e[1] != _ONE:
        raise PcpError(-1, "coef must be an f32 scalar")
    device = _one_device(g, p, v if velocities is not None else None, c, e)
    ctx = ctx or default_context(max(device, 0))
    a = NesterovManyArgs()
    with call_scope.of_described(ctx, stream, device, params, velocities or (), grads, copies or (), scale) as handle:
        a.n_tensors, a.counts, a.params, a.grads, a.dtypes = len(grads), g[1], p[0], g[0], g[2]
        a.velocities = v if velocities is None else v[0]
        if c is not None:
            a.param_copies = c[0]
        if coef is not None:
            a.coef = memoryview(e[0]).cast("q")[0]
        a.learning_rate, a.momentum, a.mode = learning_rate, momentum, int(mode)
        a.flags = 0 if sync else FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_nesterov_update_many(ctx.handle, ctypes.byref(a)), ctx.handle)


class Nesterov:
    """The reference's Nesterov optimizer (src/optimizers/nesterov.zig) with its
    velocities in HBM: init + initParameters -> __init__, update(index, param, grad),
    resetVelocity -> reset, serialize / deserialize; update_flat runs every tensor of a
    flat parameter buffer in one launch."""

    def __init__(self, counts, learning_rate: float = 0.01, momentum: float = 0.9,
                 mode: int = NesterovMode.sutskever, ctx: Context | None = None, device: int = 0):
        self.ctx = ctx or default_context(device)
        self.counts = [int(c) for c in counts]
        arr = (ctypes.c_int64 * len(self.counts))(*self.counts)
        h = ctypes.c_void_p()
        check(lib().pcp_nesterov_create(self.ctx.handle, float(learning_rate), float(momentum), int(mode),
                                        len(self.counts), arr, ctypes.byref(h)), self.ctx.handle)
        self.handle = h
        self.learning_rate, self.momentum, self.mode = float(learning_rate), float(momentum), int(mode)

    @property
    def total(self) -> int:
        return int(lib().pcp_nesterov_total(self.handle))

    def update(self, index: int, param: torch.Tensor, grad: torch.Tensor, stream=None) -> None:
        _f32(param, grad)
        check(lib().pcp_nesterov_update(self.handle, int(index), _ptr(param), _ptr(grad), param.numel(),
                                        _stream_handle(stream)), self.ctx.handle)

    def update_flat(self, params: torch.Tensor, grads: torch.Tensor, param_bf16: torch.Tensor | None = None,
                    stream=None) -> None:
        _f32(params, grads)
        if params.numel() != self.total or grads.numel() != self.total:
            raise PcpError(-12, f"flat buffers must hold {self.total} elements")
        if param_bf16 is not None and (param_bf16.dtype != torch.bfloat16 or param_bf16.numel() != self.total):
            raise PcpError(-2, "param_bf16 must be bf16 with one element per parameter")
        check(lib().pcp_nesterov_update_flat(self.handle, _ptr(params), _ptr(grads), _ptr(param_bf16),
                                             _stream_handle(stream)), self.ctx.handle)

    def update_many(self, params, grads, param_copies=None, *, coef: torch.Tensor | None = None, sync: bool = True,
                    stream=None) -> None:
        """``nesterov_update_many`` with this optimizer's velocities: params and grads in the order of its counts."""
        params, grads = list(params), list(grads)
        copies = None if param_copies is None else list(param_copies)
        if [t.numel() for t in grads] != self.counts:
            raise PcpError(-12, "the gradients must have the sizes of the optimizer's tensors")
        v = [lib().pcp_nesterov_velocity(self.handle, i) or 0 for i in range(len(self.counts))]
        _update_many(self.ctx, params, array.array("Q", v).tobytes(), None, grads, copies, coef, self.learning_rate,
                     self.momentum, self.mode, sync, stream)

    def reset(self) -> None:
        check(lib().pcp_nesterov_reset(self.handle, None), self.ctx.handle)

    def serialize(self) -> bytes:
        buf = np.empty(self.total, np.float32)
        check(lib().pcp_nesterov_serialize(self.handle, buf.ctypes.data if buf.size else None, buf.nbytes),
              self.ctx.handle)
        return buf.tobytes()

    def deserialize(self, data: bytes) -> None:
        raw = np.frombuffer(data, np.uint8) if len(data) else np.zeros(1, np.uint8)
        check(lib().pcp_nesterov_deserialize(self.handle, raw.ctypes.data, len(data)), self.ctx.handle)

    def close(self) -> None:
        if getattr(self, "handle", None):
            lib().pcp_nesterov_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _f32(*ts):
    for t in ts:
        if t.dtype != torch.float32:
            raise PcpError(-2, "parameters and gradients must be f32")


def sample_tokens(logits: torch.Tensor, temperature: float, uniforms: torch.Tensor | None = None, *,
                  ids: torch.Tensor | None = None, stream=None, ctx: Context | None = None,
                  sync: bool = True) -> torch.Tensor:
    """Sampler.sample (src/core/math.zig:21-58) on every row of logits [R, V] (f32 or
    bf16, HBM): greedy when temperature < 1e-6, else inverse-transform sampling with
    the caller's uniform draws (f32 [R] in [0, 1)). Returns int64 [R] token ids.
    sync=False only enqueues the launch on the stream (pcp_sample_tokens_async): the ids
    are ready in stream order, and ctx.sync() waits for them."""
    from ._lib import DType
    if logits.dim() != 2:
        raise PcpError(-1, "logits must be [rows, vocab]")
    code = {torch.float32: DType.f32, torch.bfloat16: DType.bf16}.get(logits.dtype)
    if code is None:
        raise PcpError(-2, "logits must be f32 or bf16")
    if logits.stride(1) != 1:
        raise PcpError(-1, "logits rows must be contiguous")
    R, V = logits.shape
    ctx = ctx or default_context(logits.device.index or 0)
    if ids is None:
        ids = torch.empty(R, dtype=torch.int64, device=logits.device)
    if uniforms is not None and (uniforms.dtype != torch.float32 or uniforms.numel() != R):
        raise PcpError(-1, "uniforms must be f32 with one value per row")
    fn = lib().pcp_sample_tokens if sync else lib().pcp_sample_tokens_async
    check(fn(ctx.handle, logits.data_ptr(), int(code), R, V, logits.stride(0), float(temperature), _ptr(uniforms),
             _ptr(ids), _stream_handle(stream)), ctx.handle)
    return ids


@dataclass
class Verified:
    tokens: torch.Tensor      # int64 [S, n + 1]: accepted tokens, the one after, IGNORE_INDEX
    accepted: torch.Tensor    # int32 [S]
    logp: torch.Tensor        # f32 [S, n + 1]: the target's log-probs of those tokens, 0 past them


def verify_drafts(target_logits: torch.Tensor, draft_ids: torch.Tensor, draft_logits: torch.Tensor | None = None, *,
                  temperature: float = 1.0, uniforms: torch.Tensor | None = None,
                  draft_lens: torch.Tensor | None = None, outputs: Verified | None = None, sync: bool = True,
                  stream=None, ctx: Context | None = None) -> Verified:
    """Speculative decoding's check of drafted tokens draft_ids [S, n] (int64) against the
    target's logits [S, n + 1, V] (f32, bf16 or f16; pcp_verify_drafts): the longest accepted
    prefix and one more token. draft_logits [S, n, V] is the distribution the tokens were drawn
    from, None for drafts looked up or chosen greedily; uniforms f32 [S, n + 1] in [0, 1), n
    for the tokens and the last for the one after (None when temperature < 1e-6, which is
    greedy); draft_lens int32 [S] the tokens drafted per sequence (None: n). The logits may be views
    with contiguous rows, such as ``logits[:, -(n + 1):]`` or a stack [n, S, V] of drafting steps,
    transposed. sync=False only enqueues the launches."""
    if target_logits.dim() != 3 or target_logits.shape[1] < 1:
        raise PcpError(-1, "target_logits must be [S, n + 1, V]")
    S, n1, V = target_logits.shape
    n = n1 - 1
    if draft_ids.shape != (S, n) or draft_ids.dtype != torch.int64:
        raise PcpError(-1, "draft_ids must be int64 [S, n]")
    if draft_logits is not None and (draft_logits.shape != (S, n, V) or draft_logits.dtype != target_logits.dtype):
        raise PcpError(-1, "draft_logits must be [S, n, V] of the target's dtype")
    if uniforms is not None and (uniforms.dtype != torch.float32 or uniforms.shape != (S, n1)):
        raise PcpError(-1, "uniforms must be f32 [S, n + 1]")
    if draft_lens is not None and (draft_lens.dtype != torch.int32 or draft_lens.shape != (S,)):
        raise PcpError(-1, "draft_lens must be int32 [S]")
    target_stride, target_seq = _row_stride(target_logits), _seq_stride(target_logits)
    draft_stride, draft_seq = (V, 0) if draft_logits is None else (_row_stride(draft_logits), _seq_stride(draft_logits))
    ctx = ctx or default_context(target_logits.device.index or 0)
    a = VerifyArgs()
    lib().pcp_verify_args_init(ctypes.byref(a))
    given = () if outputs is None else (outputs.tokens, outputs.accepted, outputs.logp)
    with call_scope(ctx, stream, target_logits, draft_ids, draft_logits, uniforms, draft_lens, *given) as handle:
        if outputs is None:
            dev = target_logits.device
            outputs = Verified(torch.empty((S, n1), dtype=torch.int64, device=dev),
                               torch.empty(S, dtype=torch.int32, device=dev),
                               torch.empty((S, n1), dtype=torch.float32, device=dev))
        o = outputs
        if (o.tokens.dtype != torch.int64 or o.tokens.numel() != S * n1 or o.accepted.dtype != torch.int32
                or o.accepted.numel() != S or o.logp.dtype != torch.float32 or o.logp.numel() != S * n1):
            raise PcpError(-1, "outputs do not fit the call: tokens int64 and logp f32 [S, n + 1], accepted int32 [S]")
        a.n_seq, a.n_draft, a.vocab = S, n, V
        a.target_row_stride, a.draft_row_stride = target_stride, draft_stride
        a.target_seq_stride, a.draft_seq_stride = target_seq, draft_seq
        a.logits_dtype, a.temperature = dtype_code(target_logits), temperature
        a.target_logits = target_logits.data_ptr()
        a.draft_logits = draft_logits.data_ptr() if draft_logits is not None and n else None
        a.draft_ids, a.draft_lens, a.uniforms = _ptr(draft_ids), _ptr(draft_lens), _ptr(uniforms)
        a.tokens, a.accepted, a.logp = _ptr(o.tokens), _ptr(o.accepted), _ptr(o.logp)
        a.flags = 0 if sync else FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_verify_drafts(ctx.handle, ctypes.byref(a)), ctx.handle)
    return outputs


def _row_stride(t: torch.Tensor) -> int:
    """Elements between the rows of a sequence of [S, m, V]."""
    _, m, V = t.shape
    _, row, one = t.stride()
    if one != 1 and V > 1:
        raise PcpError(-1, "logits rows must be contiguous")
    if m <= 1:
        return V
    if row < V:
        raise PcpError(-1, "logits rows overlap: expand them with .contiguous()")
    return row


def _seq_stride(t: torch.Tensor) -> int:
    """Elements between the sequences of [S, m, V]; 0: m rows (there is one sequence, or no row)."""
    S, m, V = t.shape
    if S <= 1 or m < 1:
        return 0
    seq = t.stride(0)
    if seq < V:
        raise PcpError(-1, "logits rows overlap: expand them with .contiguous()")
    return seq
