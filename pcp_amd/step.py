"""Device-resident work around the loss head in one training step (include/pcp_step.h):
rollout packing, gradient statistics and the Nesterov update, over torch tensors in HBM.

Mirrors RLShepherd.trainStep (src/nodes/controllers/rl_shepherd.zig:487-515 packing,
:600-641 statistics, :643-682 update loop) and the host optimizer
(src/optimizers/nesterov.zig); the arithmetic runs in libpcp_grpo.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np
import torch

from ._lib import FLAG_ASYNC, GradStats, NesterovMode, PcpError, VerifyArgs, check, lib
from .grpo import Context, _ptr, _stream_handle, call_scope, default_context, dtype_code


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
