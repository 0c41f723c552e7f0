"""Refusals of the token scores, the gradient clipping and the update of many tensors that need no GPU, their
argument structs and defaults, and the 64-bit reference's gradient against differences."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from pcp_amd import _lib, scores, step
from pcp_amd._lib import DType, PcpError
from score_ref import entropy_of, grad_ref, score_ref, softmax_parts

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")


@pytest.mark.parametrize("cname,pyty,header", [("pcp_score_args", _lib.ScoreArgs, "pcp_score.h"),
                                               ("pcp_score_bwd_args", _lib.ScoreBwdArgs, "pcp_score.h"),
                                               ("pcp_grad_clip_args", _lib.GradClipArgs, "pcp_step.h"),
                                               ("pcp_nesterov_many_args", _lib.NesterovManyArgs, "pcp_step.h")])
def test_struct_layout_matches_c(tmp_path, cname, pyty, header):
    fields = [f[0] for f in pyty._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){",
           f'printf("%zu\\n", sizeof({cname}));']
    src += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields]
    src += ["return 0;}"]
    c = tmp_path / "layout.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", INCLUDE, str(c), "-o", str(exe)], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(pyty)
    for f, off in zip(fields, vals[1:]):
        assert getattr(pyty, f).offset == off, f


def test_exported_and_limits(tmp_path):
    L = _lib.lib()
    for n in ("pcp_score_fwd", "pcp_score_bwd", "pcp_grad_clip", "pcp_nesterov_update_many", "pcp_nesterov_velocity"):
        assert n in _lib.SIGNATURES and getattr(L, n)
    c = tmp_path / "limits.c"
    c.write_text('#include <stdio.h>\n#include "pcp_score.h"\n#include "pcp_step.h"\n'
                 'int main(void){printf("%d %d", PCP_SCORE_TOP_MAX, PCP_GRAD_MAX_TENSORS);return 0;}')
    exe = tmp_path / "limits"
    subprocess.run(["gcc", "-std=c99", "-I", INCLUDE, str(c), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == [_lib.SCORE_TOP_MAX, _lib.GRAD_MAX_TENSORS]


def test_defaults():
    a = _lib.ScoreArgs()
    _lib.lib().pcp_score_args_init(ctypes.byref(a))
    assert (a.logits_dtype, a.ids_dtype, a.mask_dtype, a.top_ids_dtype) == (DType.bf16, DType.i64, DType.f32, DType.i32)
    assert a.temperature == 1.0 and a.k == 0 and not a.logits
    b = _lib.ScoreBwdArgs()
    _lib.lib().pcp_score_bwd_args_init(ctypes.byref(b))
    assert (b.logits_dtype, b.dlogits_dtype, b.accumulate, b.temperature) == (DType.bf16, DType.bf16, 0, 1.0)
    c = _lib.GradClipArgs()
    _lib.lib().pcp_grad_clip_args_init(ctypes.byref(c))
    assert c.max_norm == float("inf") and c.norm_type == 0
    d = _lib.NesterovManyArgs()
    _lib.lib().pcp_nesterov_many_args_init(ctypes.byref(d))
    assert abs(d.learning_rate - 0.01) < 1e-9 and abs(d.momentum - 0.9) < 1e-7 and d.mode == 0
    for f in ("pcp_score_args_init", "pcp_score_bwd_args_init", "pcp_grad_clip_args_init", "pcp_nesterov_many_args_init"):
        getattr(_lib.lib(), f)(None)


def filled(ty, init, **kw):
    a = ty()
    getattr(_lib.lib(), init)(ctypes.byref(a))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def fwd(**kw):
    base = dict(n_seq=2, rows=4, vocab=100, k=8, logits=0x10000, ids=0x2000, logp=0x3000, entropy=0x3100, row_max=0x3200,
                log_sum=0x3300, top_logp=0x4000, top_ids=0x5000)
    return filled(_lib.ScoreArgs, "pcp_score_args_init", **{**base, **kw})


def bwd(**kw):
    base = dict(n_seq=2, rows=4, vocab=100, logits=0x100000, ids=0x2000, row_max=0x3200, log_sum=0x3300, entropy=0x3100,
                dlogp=0x3400, dentropy=0x3500, dlogits=0x200000)
    return filled(_lib.ScoreBwdArgs, "pcp_score_bwd_args_init", **{**base, **kw})


NAN, INF = float("nan"), float("inf")
COMMON = [
    (dict(n_seq=-1), -1, "n_seq"), (dict(rows=-1), -1, "rows"), (dict(vocab=0), -1, "vocab"),
    (dict(vocab=(1 << 24) + 1), -1, "vocab"), (dict(logits_dtype=int(DType.f64)), -2, "logits dtype"),
    (dict(ids_dtype=int(DType.f32)), -2, "ids dtype"), (dict(mask=0x6000, mask_dtype=int(DType.i64)), -2, "mask dtype"),
    (dict(temperature=0.0), -1, "temperature"), (dict(temperature=-1.0), -1, "temperature"),
    (dict(temperature=NAN), -1, "temperature"), (dict(temperature=INF), -1, "temperature"),
    (dict(temperature=1e-39), -1, "temperature"), (dict(flags=2), -1, "PCP_FLAG_ASYNC"),
    (dict(tok_offset=1), -1, "tok_offset"), (dict(tok_offset=-1), -1, "tok_offset"),
    (dict(tok_offset=(1 << 63) - 1), -1, "tok_offset"), (dict(tok_seq_stride=3), -1, "tok_offset"),
    (dict(tok_seq_stride=1 << 61), -9, "token array"), (dict(logits=0x10001), -1, "element size"),
    (dict(ids=0x2004), -1, "element size"), (dict(mask=0x6002), -1, "element size"),
    (dict(row_stride=99), -1, "row_stride"), (dict(seq_stride=99), -1, "seq_stride"),
    (dict(seq_stride=1 << 61), -9, "overflows"), (dict(row_stride=1 << 61), -9, "overflows"),
    (dict(logits=None), -1, "NULL"), (dict(row_max=0x3201), -1, "element size"), (dict(entropy=0x3102), -1, "element size"),
    (dict(), -1, "context is NULL"),
]


@pytest.mark.parametrize("change,code,text", COMMON + [
    (dict(k=-1), -1, "k must"), (dict(k=257, vocab=1000), -1, "k must"), (dict(k=101), -1, "k must"),
    (dict(n_seq=1 << 30), -9, "rows"), (dict(top_ids_dtype=int(DType.f32)), -2, "top_ids dtype"),
    (dict(top_logp=None), -1, "NULL"), (dict(top_ids=None), -1, "NULL"), (dict(ids=None), -1, "logp needs ids"),
    (dict(logp=0x3001), -1, "element size"), (dict(top_ids=0x5004, top_ids_dtype=int(DType.i64)), -1, "element size"),
])
def test_fwd_refusals(change, code, text):
    L = _lib.lib()
    assert L.pcp_score_fwd(None, ctypes.byref(fwd(**change))) == code
    assert text in L.pcp_last_error(None).decode()


@pytest.mark.parametrize("change,code,text", COMMON + [
    (dict(logit_rows=3), -1, "logit_rows"), (dict(n_seq=1 << 30), -9, "rows"), (dict(logit_rows=1 << 30), -9, "rows"),
    (dict(dlogits_dtype=int(DType.f16)), -2, "dlogits dtype"), (dict(drow_stride=99), -1, "drow_stride"),
    (dict(dseq_stride=99), -1, "dseq_stride"), (dict(dseq_stride=150), -1, "rows of dlogits overlap"),
    (dict(drow_stride=150, dseq_stride=100), -1, "rows of dlogits overlap"),
    (dict(dlogits=None), -1, "dlogits is NULL"), (dict(row_max=None), -1, "NULL"), (dict(log_sum=None), -1, "NULL"),
    (dict(ids=None), -1, "dlogp needs ids"), (dict(entropy=None), -1, "entropy"),
    (dict(dlogits=0x200001), -1, "element size"), (dict(dlogp=0x3402), -1, "element size"),
    (dict(dlogits=0x100010), -1, "overlap the logits"), (dict(dlogits=0x100000, dlogits_dtype=int(DType.f32)), -1, "overlap"),
    (dict(dlogits=0x100000, drow_stride=104), -1, "overlap the logits"),
])
def test_bwd_refusals(change, code, text):
    L = _lib.lib()
    assert L.pcp_score_bwd(None, ctypes.byref(bwd(**change))) == code
    assert text in L.pcp_last_error(None).decode()


def test_bwd_allows():
    """Calls that get as far as the missing context: in place, rows of sequences between one another, no rows."""
    L = _lib.lib()
    for change in (dict(dlogits=0x100000), dict(drow_stride=200, dseq_stride=100), dict(dlogp=None, ids=None),
                   dict(dentropy=None, entropy=None), dict(rows=0, logit_rows=4, logits=None, row_max=None, log_sum=None),
                   dict(n_seq=0, dlogits=None, logits=None)):
        assert L.pcp_score_bwd(None, ctypes.byref(bwd(**change))) == -1
        assert "context is NULL" in L.pcp_last_error(None).decode(), change


def lists(n, **columns):
    keep = {}
    for name, vals in columns.items():
        ty = ctypes.c_int64 if name == "counts" else ctypes.c_int32 if name.endswith("dtypes") else ctypes.c_void_p
        keep[name] = (ty * n)(*vals)
    return keep


CLIP = dict(grads=[0x10000, 0x20000], counts=[100, 50], dtypes=[2, 1], out=[0x30000, 0x40000], out_dtypes=[2, 2])
NEST = dict(counts=[100, 50], params=[0x10000, 0x20000], velocities=[0x30000, 0x40000], grads=[0x50000, 0x60000],
            dtypes=[2, 1], param_copies=[0x70000, 0])


def call_list(ty, init, fn, base, plain, change):
    cols = {**base, **{k: v for k, v in change.items() if k in base}}
    n = 2
    keep = lists(n, **{k: v for k, v in cols.items() if v is not None})
    a = filled(ty, init, **plain)
    a.n_tensors = n
    for k, v in keep.items():
        setattr(a, k, ctypes.addressof(v))
    for k, v in change.items():
        if k not in base:
            setattr(a, k, v)
    L = _lib.lib()
    return getattr(L, fn)(None, ctypes.byref(a)), L.pcp_last_error(None).decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(n_tensors=-1), -1, "n_tensors"), (dict(n_tensors=262145), -1, "n_tensors"), (dict(counts=[-1, 5]), -1, "counts[0]"),
    (dict(counts=[1 << 43, 1 << 44]), -9, "2^44"), (dict(counts=None), -1, "counts is NULL"),
    (dict(norm_type=2), -1, "norm_type"), (dict(max_norm=0.0), -1, "max_norm"), (dict(max_norm=-1.0), -1, "max_norm"),
    (dict(max_norm=NAN), -1, "max_norm"), (dict(flags=4), -1, "PCP_FLAG_ASYNC"), (dict(norm=None), -1, "NULL"),
    (dict(coef=None), -1, "NULL"), (dict(grads=None), -1, "NULL"), (dict(grads=[0, 0x20000]), -1, "tensor 0 is NULL"),
    (dict(out=[0x30000, 0]), -1, "tensor 1 is NULL"), (dict(dtypes=[3, 1]), -2, "types"), (dict(out_dtypes=[2, 4]), -2, "types"),
    (dict(grads=[0x10002, 0x20000]), -1, "element size"), (dict(out=[0x30000, 0x40002]), -1, "element size"),
    (dict(norm=0x1002), -1, "element size"),
    (dict(out=[0x30000, 0x30000]), -1, "overlaps"),                      # two outputs in one place
    (dict(out=[0x10000, 0x10000], out_dtypes=[2, 2]), -1, "overlaps"),
    (dict(out=[0x10004, 0x40000]), -1, "overlaps"),                      # an output beside its gradient's place
    (dict(out=[0x20000, 0x40000]), -1, "overlaps"),                      # over another gradient
    (dict(out=[0x30000, 0x20000]), -1, "overlaps"),                      # in place in another type
    (dict(grads=[0x10000, 0x10000], dtypes=[2, 2], out=[0x10000, 0x10000]), -1, "overlaps"),   # one gradient twice
    (dict(norm=0x10004, out=[0x10000, 0x40000]), -1, "overlaps"),
    (dict(), -1, "context is NULL"), (dict(out=None, grads=[0x10000, 0x10000]), -1, "context is NULL"),
    (dict(out=[0x10000, 0x40000]), -1, "context is NULL"), (dict(grads=[0, 0x20000], out=[0, 0x40000], counts=[0, 50]), -1, "context is NULL"),
])
def test_clip_refusals(change, code, text):
    got, said = call_list(_lib.GradClipArgs, "pcp_grad_clip_args_init", "pcp_grad_clip", CLIP,
                          dict(norm=0x1000, coef=0x1004, max_norm=1.0), change)
    assert got == code and text in said, said


@pytest.mark.parametrize("change,code,text", [
    (dict(n_tensors=-1), -1, "n_tensors"), (dict(counts=[5, -2]), -1, "counts[1]"), (dict(mode=2), -1, "mode"),
    (dict(learning_rate=NAN), -1, "finite"), (dict(momentum=INF), -1, "finite"), (dict(flags=2), -1, "PCP_FLAG_ASYNC"),
    (dict(params=None), -1, "NULL"), (dict(velocities=None), -1, "NULL"), (dict(grads=None), -1, "NULL"),
    (dict(params=[0x10000, 0]), -1, "tensor 1 is NULL"), (dict(dtypes=[2, 5]), -2, "gradients must be"),
    (dict(params=[0x10002, 0x20000]), -1, "element size"), (dict(param_copies=[0x70001, 0]), -1, "element size"),
    (dict(coef=0x1001), -1, "element size"), (dict(params=[0x10000, 0x10000]), -1, "overlaps"),
    (dict(velocities=[0x10000, 0x40000]), -1, "overlaps"), (dict(grads=[0x10000, 0x60000]), -1, "overlaps"),
    (dict(param_copies=[0x50000, 0]), -1, "overlaps"), (dict(coef=0x10004), -1, "overlaps"),
    (dict(), -1, "context is NULL"), (dict(grads=[0x50000, 0x50000]), -1, "context is NULL"),
])
def test_update_refusals(change, code, text):
    got, said = call_list(_lib.NesterovManyArgs, "pcp_nesterov_many_args_init", "pcp_nesterov_update_many", NEST,
                          dict(coef=0x1000), change)
    assert got == code and text in said, said


def test_null_args():
    L = _lib.lib()
    for fn in ("pcp_score_fwd", "pcp_score_bwd", "pcp_grad_clip", "pcp_nesterov_update_many"):
        assert getattr(L, fn)(None, None) == -1
        assert "args is NULL" in L.pcp_last_error(None).decode()
    assert L.pcp_nesterov_velocity(None, 0) is None


def test_python_refusals():
    x, ids = torch.zeros(2, 4, 10), torch.zeros(2, 4, dtype=torch.int64)
    f = torch.zeros(2, 4)
    for call in (lambda: scores.token_scores(x[0], ids), lambda: scores.token_scores(x, ids[0]),
                 lambda: scores.token_scores(x, ids, torch.zeros(2, 5)), lambda: scores.token_scores(x, ids, k=11),
                 lambda: scores.token_scores(x, ids, k=-1), lambda: scores.token_scores(x, ids, rows=5),
                 lambda: scores.token_scores(x, ids, tok_offset=1), lambda: scores.token_scores(x, tokens=3),
                 lambda: scores.token_scores(x.transpose(1, 2), torch.zeros(2, 10, dtype=torch.int64)),
                 lambda: scores.token_scores(x[:, :1].expand(2, 4, 10), ids),
                 lambda: scores.token_scores_bwd(x, ids, f, f[:1]), lambda: scores.token_scores_bwd(x, None, f, f, dlogp=f),
                 lambda: scores.token_scores_bwd(x, ids, f, f, dentropy=f),
                 lambda: scores.token_scores_bwd(x, ids, f, f, accumulate=True),
                 lambda: scores.token_scores_bwd(x, ids, f, f.double()),
                 lambda: scores.token_scores_bwd(x, ids, f, f, dlogits=x[:, :, :9]),
                 lambda: scores.token_scores_bwd(x, ids, f, f, dlogits=x, dlogits_dtype=torch.bfloat16),
                 lambda: step.grad_norm([f], norm_type="l1", outputs=step.GradNorm(f[0, 0], f[0, 1])),
                 lambda: step.nesterov_update_many([f], [f], [f], mode="adam")):
        with pytest.raises(PcpError):
            call()


@pytest.mark.parametrize("tau", [1.0, 0.5, 2.0])
def test_reference_gradient_against_differences(tau):
    """d (gl logp + gh entropy) / dx by central differences; and that the parts agree with one another."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 9)) * 2
    x[1, 4] = -np.inf
    ids, gl, gh = np.array([2, 0, 8]), np.array([0.7, -1.1, 0.0]), np.array([-0.3, 0.4, 1.5])

    def f(x):
        logp, h, *_ = score_ref(x, ids, tau)
        return gl @ logp + gh @ h

    g, bar = grad_ref(x, ids, gl, gh, tau)
    assert (bar >= 0).all() and abs(g.sum()) < 1e-12   # a shift of a row changes nothing
    for r, v in np.ndindex(x.shape):
        if not np.isfinite(x[r, v]):
            assert g[r, v] == 0
            continue
        hi, lo = x.copy(), x.copy()
        hi[r, v] += 1e-5
        lo[r, v] -= 1e-5
        assert abs((f(hi) - f(lo)) / 2e-5 - g[r, v]) < 1e-8
    m, log_sum, log_p = softmax_parts(x, tau)
    assert np.allclose(np.exp(log_p).sum(1), 1) and (entropy_of(log_p) <= np.log(9) + 1e-12).all()


def test_overlaps_are_found_in_any_order():
    """Random lists of ranges, rising or shuffled, against every pair of them."""
    rng = np.random.default_rng(11)
    L = _lib.lib()
    seen = set()
    for turn in range(400):
        n = int(rng.integers(1, 6))
        counts = rng.integers(0, 6, n)
        room = int(rng.choice([60, 400, 4000]))
        cols = {k: rng.integers(1, room, n) * 4 + 0x1000 for k in ("params", "velocities", "grads", "param_copies")}
        if turn % 2:                                       # pieces of flat buffers, at times one over another
            base = 0x1000
            for k in cols:
                cols[k] = base + np.concatenate([[0], np.cumsum(counts[:-1])]) * 4
                base += int(counts.sum()) * 4 - (8 if rng.random() < 0.2 else 0)
        size = {"params": 4, "velocities": 4, "grads": 4, "param_copies": 2}
        spans = [(int(cols[k][i]), int(cols[k][i]) + int(counts[i]) * size[k], k != "grads")
                 for k in cols for i in range(n) if counts[i]]
        meet = any(a[0] < b[1] and b[0] < a[1] and (a[2] or b[2]) for i, a in enumerate(spans) for b in spans[:i])
        keep = lists(n, counts=[int(c) for c in counts], **{k: [int(x) for x in v] for k, v in cols.items()})
        a = filled(_lib.NesterovManyArgs, "pcp_nesterov_many_args_init")
        a.n_tensors = n
        for k, v in keep.items():
            setattr(a, k, ctypes.addressof(v))
        assert L.pcp_nesterov_update_many(None, ctypes.byref(a)) == -1
        assert ("overlaps" if meet else "context is NULL") in L.pcp_last_error(None).decode(), (spans, meet)
        seen.add((turn % 2, meet))
    assert len(seen) == 4
