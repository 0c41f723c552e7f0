"""Learning from another model's distribution (include/pcp_distill.h) over torch tensors in
HBM: the top logits of a teacher's rows, and the distillation loss on them with its gradient.

The reference trains by GRPO alone; rows, masks and the aggregation of the loss are those of
``pcp_amd.grpo`` (logits [S, LS, V], token arrays [S, TS], row (s, t) weighted by
mask[s, tok_offset + t]). The arithmetic runs in libpcp_grpo.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import DistillArgs, Divergence, PcpError, TopLogitsArgs, check, lib
from .grpo import Context, _ptr, call_scope, default_context, dtype_code


@dataclass
class TopLogits:
    values: torch.Tensor          # f32 [..., k], falling
    ids: torch.Tensor             # i32 / i64 [..., k]
    lse: torch.Tensor             # f32 [...]: log sum exp(logits / temperature)


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0, ids_dtype: torch.dtype = torch.int32,
               outputs: TopLogits | None = None, sync: bool = True, stream=None,
               ctx: Context | None = None) -> TopLogits:
    """The k largest logits of every row of logits [..., V] (f32, bf16 or f16) with their
    ids (equal logits by rising id), and each row's log-sum-exp at `temperature`
    (pcp_top_logits). A [R, V] view may have rows further apart than V. Pass ``outputs``
    of an earlier call of the same shape to reuse its buffers; sync=False only enqueues."""
    if logits.dim() < 1 or logits.stride(-1) != 1:
        raise PcpError(-1, "logits must be [..., vocab] with contiguous rows")
    if not logits.is_contiguous() and logits.dim() != 2:
        raise PcpError(-1, "logits of more than two dimensions must be contiguous")
    V = logits.shape[-1]
    R = logits.numel() // V if V else 0
    if logits.dim() == 2 and R > 1 and logits.stride(0) < V:
        raise PcpError(-1, "logits rows overlap: expand them with .contiguous()")
    k = int(k)
    if not 1 <= k <= min(V, _lib.TOP_LOGITS_MAX):
        raise PcpError(-1, f"k must be in [1, {min(V, _lib.TOP_LOGITS_MAX)}] (got {k})")
    ctx = ctx or default_context(logits.device.index or 0)
    a = TopLogitsArgs()
    lib().pcp_top_logits_args_init(ctypes.byref(a))
    given = () if outputs is None else (outputs.values, outputs.ids, outputs.lse)
    with call_scope(ctx, stream, logits, *given) as handle:
        if outputs is None:
            lead, dev = tuple(logits.shape[:-1]), logits.device
            outputs = TopLogits(torch.empty(lead + (k,), dtype=torch.float32, device=dev),
                                torch.empty(lead + (k,), dtype=ids_dtype, device=dev),
                                torch.empty(lead, dtype=torch.float32, device=dev))
        o = outputs
        if (o.values.dtype != torch.float32 or o.values.numel() != R * k or o.ids.dtype != ids_dtype
                or o.ids.numel() != R * k or o.lse.dtype != torch.float32 or o.lse.numel() != R):
            raise PcpError(-1, "outputs do not fit the call: values f32 and ids [rows, k], lse f32 [rows]")
        a.n_rows, a.vocab, a.k = R, V, k
        a.row_stride = logits.stride(0) if logits.dim() == 2 and R > 1 else V
        a.logits_dtype, a.ids_dtype, a.temperature = dtype_code(logits), dtype_code(o.ids), temperature
        a.logits, a.values, a.ids, a.lse = logits.data_ptr(), _ptr(o.values), _ptr(o.ids), _ptr(o.lse)
        a.flags = 0 if sync else _lib.FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_top_logits(ctx.handle, ctypes.byref(a)), ctx.handle)
    return outputs


@dataclass
class DistillOutputs:
    loss: torch.Tensor            # f32 scalar
    token_loss: torch.Tensor      # f32 [S, TS]
    dlogits: torch.Tensor | None  # [S, LS, V]


def distill_fwd_bwd(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                    teacher_lse: torch.Tensor | None = None, mask: torch.Tensor | None = None, *,
                    divergence: int | str = Divergence.forward, temperature: float = 1.0, weight: float = 1.0,
                    loss_norm: float = 0.0, rows: int | None = None, tok_offset: int = 0, tokens: int | None = None,
                    want_dlogits: bool = True, dlogits: torch.Tensor | None = None,
                    dlogits_dtype: torch.dtype | None = None, outputs: DistillOutputs | None = None,
                    sync: bool = True, stream=None, ctx: Context | None = None) -> DistillOutputs:
    """Distillation loss of the student's logits [S, LS, V] against a teacher's entries
    teacher_ids / teacher_logits [S, LS, k] (as ``top_logits`` of the teacher's [S, LS, V]
    returns them) and its dlogits (pcp_distill_fwd_bwd).

    With teacher_lse [S, LS] (at the same temperature) the teacher's other tokens are one
    more class; without, its entries are renormalised. divergence is "forward"
    (sum p log(p/q)) or "reverse" (sum q log(q/p), which needs teacher_lse). An id of
    IGNORE_INDEX leaves an entry unused. mask [S, TS] weights tokens as in
    ``grpo_loss_fwd_bwd``; without a mask, `tokens` (default LS) is TS.

    dlogits is written into `dlogits` or, with ``outputs`` of an earlier call, into theirs (one
    of the two; dlogits_dtype only says what a new one holds). want_dlogits=False forms the
    loss alone and leaves ``outputs.dlogits`` as it is."""
    if logits.dim() != 3:
        raise PcpError(-1, "logits must be [S, LS, V]")
    S, LS, V = logits.shape
    if teacher_ids.dim() != 3 or teacher_ids.shape[:2] != logits.shape[:2] or teacher_logits.shape != teacher_ids.shape:
        raise PcpError(-1, "teacher_ids and teacher_logits must both be [S, LS, k]")
    if teacher_logits.dtype != torch.float32:
        raise PcpError(-2, "teacher_logits must be f32")
    if teacher_lse is not None and (teacher_lse.dtype != torch.float32 or teacher_lse.shape != logits.shape[:2]):
        raise PcpError(-1, "teacher_lse must be f32 [S, LS]")
    if mask is not None and (mask.dim() != 2 or mask.shape[0] != S):
        raise PcpError(-1, "mask must be [S, TS]")
    if isinstance(divergence, str):
        try:
            divergence = Divergence[divergence]
        except KeyError:
            raise PcpError(-1, f"unknown divergence {divergence!r}") from None
    if dlogits is not None and not want_dlogits:
        raise PcpError(-1, "dlogits is given and want_dlogits is False")
    if outputs is not None and dlogits is not None and dlogits is not outputs.dlogits:
        raise PcpError(-1, "dlogits is given twice: by itself and in outputs")
    if want_dlogits and dlogits_dtype is not None:
        into = dlogits if outputs is None else outputs.dlogits
        if into is not None and into.dtype != dlogits_dtype:
            raise PcpError(-2, f"dlogits_dtype is {dlogits_dtype}, the given dlogits are {into.dtype}")
        if into is None and outputs is not None:
            raise PcpError(-1, "dlogits_dtype is given and outputs have no dlogits")
    TS = mask.shape[1] if mask is not None else (LS if tokens is None else int(tokens))
    rows, tok_offset = LS if rows is None else int(rows), int(tok_offset)
    # (A mask or token count of no tokens has no pointer and no stride: the C entry would take it for
    # "no mask" and "one token per row".)
    if rows < 0 or tok_offset < 0 or tok_offset + rows > TS:
        raise PcpError(-1, f"{rows} rows from token {tok_offset} on do not fit in {TS} tokens")
    if not 1 <= teacher_ids.shape[2] <= _lib.TOP_LOGITS_MAX:
        raise PcpError(-1, f"k must be in [1, {_lib.TOP_LOGITS_MAX}] (got {teacher_ids.shape[2]})")
    ctx = ctx or default_context(logits.device.index or 0)
    a = DistillArgs()
    lib().pcp_distill_args_init(ctypes.byref(a))
    given = (dlogits,) if outputs is None else (outputs.loss, outputs.token_loss, outputs.dlogits)
    with call_scope(ctx, stream, logits, teacher_ids, teacher_logits, teacher_lse, mask, *given) as handle:
        if outputs is None:
            dev = logits.device
            if want_dlogits and dlogits is None:
                dlogits = torch.empty((S, LS, V), dtype=dlogits_dtype or logits.dtype, device=dev)
            outputs = DistillOutputs(torch.empty((), dtype=torch.float32, device=dev),
                                     torch.zeros((S, TS), dtype=torch.float32, device=dev),
                                     dlogits)
        o = outputs
        if (o.loss.dtype != torch.float32 or o.loss.numel() != 1 or o.token_loss.dtype != torch.float32
                or o.token_loss.numel() != S * TS or (o.dlogits is not None and o.dlogits.numel() != S * LS * V)):
            raise PcpError(-1, "outputs do not fit the call: loss f32 [], token_loss f32 [S, TS], dlogits [S, LS, V]")
        a.n_seq, a.rows, a.vocab = S, rows, V
        a.logit_seq_stride, a.tok_seq_stride, a.tok_offset = LS, TS, tok_offset
        a.k, a.divergence = teacher_ids.shape[2], int(divergence)
        a.logits_dtype, a.ids_dtype = dtype_code(logits), dtype_code(teacher_ids)
        a.logits, a.teacher_ids, a.teacher_logits = _ptr(logits), _ptr(teacher_ids), _ptr(teacher_logits)
        a.teacher_lse = _ptr(teacher_lse)
        if mask is not None:
            a.mask, a.mask_dtype = _ptr(mask), dtype_code(mask)
        if o.dlogits is not None and want_dlogits:
            a.dlogits, a.dlogits_dtype = _ptr(o.dlogits), dtype_code(o.dlogits)
        a.token_loss, a.loss = _ptr(o.token_loss), _ptr(o.loss)
        a.temperature, a.weight, a.loss_norm = temperature, weight, loss_norm
        a.flags = 0 if sync else _lib.FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_distill_fwd_bwd(ctx.handle, ctypes.byref(a)), ctx.handle)
    return outputs
