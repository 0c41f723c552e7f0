"""Scores of given tokens over torch tensors in HBM (include/pcp_score.h): log-probs, entropy and the top
alternatives of rows of logits, and the gradient of any function of the log-probs and entropies.

The reference scores tokens inside its training graph alone (tools/export_qwen_forward.py:154-156). Token
arrays, masks and the shifted layout are those of ``pcp_amd.grpo``; the arithmetic runs in libpcp_grpo.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import DType, PcpError, ScoreArgs, ScoreBwdArgs, check, lib
from .grpo import _TORCH_DTYPE, Context, call_scope, default_context, dtype_code

_F32 = int(DType.f32)
_NO_FIT = "outputs do not fit the call: f32 [S, TS], top_logp f32 and top_ids [S, TS, k]"


@dataclass
class TokenScores:
    logp: torch.Tensor | None      # f32 [S, TS]; None without ids
    entropy: torch.Tensor          # f32 [S, TS]
    row_max: torch.Tensor          # f32 [S, TS]: the row's largest logit
    log_sum: torch.Tensor          # f32 [S, TS]: log sum exp((x - row_max) / temperature)
    top_logp: torch.Tensor | None  # f32 [S, TS, k], falling; None where k is 0
    top_ids: torch.Tensor | None   # i32 / i64 [S, TS, k]


def _tokens(logits, ids, mask, rows, tok_offset, tokens):
    """(S, LS, V, TS, rows, tok_offset) of a call on logits [S, LS, V]."""
    if logits.dim() != 3:
        raise PcpError(-1, "logits must be [S, LS, V]")
    S, LS, V = logits.shape
    TS = LS if tokens is None else int(tokens)
    for t, name in ((mask, "mask"), (ids, "ids")):
        if t is not None:
            if t.dim() != 2 or t.shape[0] != S:
                raise PcpError(-1, f"{name} must be [S, TS]")
            TS = t.shape[1]
    if ids is not None and mask is not None and ids.shape != mask.shape:
        raise PcpError(-1, "ids and mask must have the same shape")
    rows, tok_offset = LS if rows is None else int(rows), int(tok_offset)
    if rows < 0 or rows > LS:
        raise PcpError(-1, f"{rows} rows of sequences of {LS}")
    # (Token arrays of no tokens have no pointer and no stride: the C entry would take them for absent ones.)
    if tok_offset < 0 or tok_offset + rows > TS:
        raise PcpError(-1, f"{rows} rows from token {tok_offset} on do not fit in {TS} tokens")
    return S, LS, V, TS, rows, tok_offset


def _row_strides(t: torch.Tensor) -> tuple[int, int]:
    """Elements between the rows and between the sequences of [S, LS, V]."""
    S, m, V = t.shape
    seq, row, one = t.stride()
    if one != 1 and V > 1:
        raise PcpError(-1, "logits rows must be contiguous")
    if m <= 1:
        row = V
    if S <= 1 or m < 1:
        seq = max(m, 1) * row
    if row < V or seq < V:
        raise PcpError(-1, "logits rows overlap: expand them with .contiguous()")
    return row, seq


def token_scores(logits: torch.Tensor, ids: torch.Tensor | None = None, mask: torch.Tensor | None = None, *, k: int = 0,
                 temperature: float = 1.0, rows: int | None = None, tok_offset: int = 0, tokens: int | None = None,
                 top_ids_dtype: torch.dtype = torch.int32, outputs: TokenScores | None = None, sync: bool = True,
                 stream=None, ctx: Context | None = None) -> TokenScores:
    """Log-probs of ids [S, TS] under logits [S, LS, V] (f32, bf16 or f16) at `temperature`, each row's entropy,
    and its k largest logits as log-probs with their ids (equal logits by rising id): pcp_score_fwd. Row (s, t),
    t < rows, scores token tok_offset + t; rows whose token weighs 0 in mask [S, TS] or is IGNORE_INDEX are
    left out (zeros, ids IGNORE_INDEX). Without ids no log-probs are formed; without a mask too, `tokens`
    (default LS) is TS. The logits may be views with contiguous rows, such as ``logits[:, -n:]``, rows of a padded
    vocabulary or a stack of decode steps [n, S, V], transposed.

    Pass ``outputs`` of an earlier call of the same shape to reuse its buffers; entries that no row addresses
    keep their values (zeros in new ones). sync=False only enqueues."""
    S, LS, V, TS, rows, tok_offset = _tokens(logits, ids, mask, rows, tok_offset, tokens)
    k = int(k)
    if not 0 <= k <= min(V, _lib.SCORE_TOP_MAX):
        raise PcpError(-1, f"k must be in [0, {min(V, _lib.SCORE_TOP_MAX)}] (got {k})")
    a = ScoreArgs()
    a.row_stride, a.seq_stride = _row_strides(logits)
    o = outputs
    if o is not None and not (_lib.fit((o.logp if ids is not None else None, o.entropy, o.row_max, o.log_sum), S, TS)
                              and (k == 0 or _lib.fit((o.top_logp, o.top_ids), S, TS, k))):
        raise PcpError(-1, _NO_FIT)
    ctx = ctx or default_context(logits.device.index or 0)
    if o is None:
        made = lambda *shape: torch.zeros(shape, dtype=torch.float32, device=logits.device)  # noqa: E731
    given = () if o is None else (o.logp if ids is not None else None, o.entropy, o.row_max, o.log_sum,
                                  o.top_logp if k else None, o.top_ids if k else None)
    known = (ids, mask, *given)
    d = _lib.describe((logits, *known))
    _contiguous(d)
    with call_scope.of_described(ctx, stream, d[4], (logits, *known)) as handle:
        if o is None:
            o = TokenScores(made(S, TS) if ids is not None else None, made(S, TS), made(S, TS), made(S, TS),
                            made(S, TS, k) if k else None,
                            torch.zeros((S, TS, k), dtype=top_ids_dtype, device=logits.device) if k else None)
            known = (ids, mask, o.logp, o.entropy, o.row_max, o.log_sum, o.top_logp, o.top_ids)
            d = _lib.describe((logits, *known))
        else:
            # (Optional ones may be None: but logp with ids, and the alternatives with k.)
            f32, top = _F32, int(_TORCH_DTYPE.get(top_ids_dtype, -2))
            n, t = memoryview(d[1]).cast("q")[3:].tolist(), memoryview(d[2]).cast("i")[3:].tolist()
            N = S * TS
            want = [N if ids is not None else -1, N, N, N, N * k if k else -1, N * k if k else -1]
            types = [f32 if ids is not None else -1, f32, f32, f32, f32 if k else -1, top if k else -1]
            if n != want or t != types:
                for i in range(6):
                    if (n[i] != want[i] or t[i] != types[i]) and not (n[i] == -1 and 1 <= i <= 3):
                        raise PcpError(-1, _NO_FIT)
        at = memoryview(d[0]).cast("q")
        a.n_seq, a.rows, a.vocab, a.tok_seq_stride, a.tok_offset = S, rows, V, TS, tok_offset
        kinds = memoryview(d[2]).cast("i")
        a.k, a.temperature, a.logits, a.ids, a.mask = k, temperature, at[0], at[1], at[2]
        a.logits_dtype, a.ids_dtype, a.mask_dtype, a.top_ids_dtype = kinds[0], kinds[1], kinds[2], kinds[8]
        a.logp, a.entropy, a.row_max, a.log_sum, a.top_logp, a.top_ids = at[3:]
        a.flags = 0 if sync else _lib.FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_score_fwd(ctx.handle, ctypes.byref(a)), ctx.handle)
    return o


def token_scores_bwd(logits: torch.Tensor, ids: torch.Tensor | None, row_max: torch.Tensor, log_sum: torch.Tensor,
                     entropy: torch.Tensor | None = None, *, dlogp: torch.Tensor | None = None,
                     dentropy: torch.Tensor | None = None, mask: torch.Tensor | None = None, temperature: float = 1.0,
                     rows: int | None = None, tok_offset: int = 0, dlogits: torch.Tensor | None = None,
                     dlogits_dtype: torch.dtype | None = None, accumulate: bool = False, sync: bool = True, stream=None,
                     ctx: Context | None = None) -> torch.Tensor:
    """dlogits [S, LS, V] of a function of ``token_scores``' logp and entropy, whose gradients are dlogp and
    dentropy [S, TS] (f32, either may be None for 0): pcp_score_bwd. row_max, log_sum and (for dentropy) entropy are
    the forward's, at the same temperature, rows and tok_offset. With accumulate the gradient is added to the
    given dlogits (the loss head's, for an entropy bonus); rows that have none stay as they are, and are 0
    otherwise. dlogits may be the logits themselves, and views with contiguous rows as the logits may."""
    S, LS, V, TS, rows, tok_offset = _tokens(logits, ids, mask, rows, tok_offset, row_max.shape[1] if row_max.dim() == 2 else 0)
    if dlogp is not None and ids is None:
        raise PcpError(-1, "dlogp needs ids")
    if dentropy is not None and entropy is None:
        raise PcpError(-1, "dentropy needs the forward's entropy")
    if dlogits is None and accumulate:
        raise PcpError(-1, "accumulate needs dlogits")
    if dlogits is not None and dlogits.shape != logits.shape:
        raise PcpError(-1, "dlogits must have the logits' shape")
    if dlogits is not None and dlogits_dtype is not None and dlogits.dtype != dlogits_dtype:
        raise PcpError(-2, f"dlogits_dtype is {dlogits_dtype}, the given dlogits are {dlogits.dtype}")
    a = ScoreBwdArgs()
    a.row_stride, a.seq_stride = _row_strides(logits)
    known = (logits, ids, mask, row_max, log_sum, entropy, dlogp, dentropy)
    if row_max is None or log_sum is None or not _lib.fit(known[3:], S, TS):
        raise PcpError(-1, "row_max, log_sum, entropy, dlogp and dentropy must be [S, TS]")
    ctx = ctx or default_context(logits.device.index or 0)
    d = _lib.describe((*known, dlogits))
    _contiguous(d, len(known))
    kinds = memoryview(d[2]).cast("i").tolist()
    if kinds[3:5] != [_F32, _F32] or any([t != _F32 and t != -1 for t in kinds[5:8]]):
        raise PcpError(-2, "row_max, log_sum, entropy, dlogp and dentropy must be f32")
    with call_scope.of_described(ctx, stream, d[4], known, (dlogits,)) as handle:
        if dlogits is None:
            dlogits = torch.empty((S, LS, V), dtype=dlogits_dtype or logits.dtype, device=logits.device)
        a.drow_stride, a.dseq_stride = _row_strides(dlogits)
        at = memoryview(d[0]).cast("q")
        a.n_seq, a.rows, a.logit_rows, a.vocab, a.tok_seq_stride, a.tok_offset = S, rows, LS, V, TS, tok_offset
        a.logits_dtype, a.ids_dtype, a.mask_dtype, a.dlogits_dtype = *kinds[:3], dtype_code(dlogits)
        a.temperature, a.logits, a.ids, a.mask, a.dlogits = temperature, at[0], at[1], at[2], dlogits.data_ptr()
        a.row_max, a.log_sum, a.entropy, a.dlogp, a.dentropy = at[3:8]
        a.accumulate = 1 if accumulate else 0
        a.flags = 0 if sync else _lib.FLAG_ASYNC
        a.stream = handle
        check(lib().pcp_score_bwd(ctx.handle, ctypes.byref(a)), ctx.handle)
    return dlogits


def _contiguous(d, n: int | None = None) -> None:
    """The first n described tensors behind the logits are contiguous."""
    if 0 in d[3][1:n]:
        raise PcpError(-1, "token arrays and outputs must be contiguous")
