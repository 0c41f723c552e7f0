"""Refusals of the distillation and draft-verification entry points that need no GPU, their
argument structs and defaults, and the 64-bit reference against differences."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from distill_ref import lse_ref, row_ref, top_ref, verify_ref
from pcp_amd import _lib, distill, step
from pcp_amd._lib import DType, PcpError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")


@pytest.mark.parametrize("cname,pyty,header", [("pcp_top_logits_args", _lib.TopLogitsArgs, "pcp_distill.h"),
                                               ("pcp_distill_args", _lib.DistillArgs, "pcp_distill.h"),
                                               ("pcp_verify_args", _lib.VerifyArgs, "pcp_sample.h")])
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


def filled(ty, init, **kw):
    a = ty()
    getattr(_lib.lib(), init)(ctypes.byref(a))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def top(**kw):
    base = dict(n_rows=2, vocab=100, k=8, logits=0x1000, values=0x2000, ids=0x3000)
    return filled(_lib.TopLogitsArgs, "pcp_top_logits_args_init", **{**base, **kw})


def dist(**kw):
    base = dict(n_seq=2, rows=4, vocab=100, k=8, logits=0x100000, teacher_ids=0x2000, teacher_logits=0x3000,
                dlogits=0x200000)
    return filled(_lib.DistillArgs, "pcp_distill_args_init", **{**base, **kw})


def ver(**kw):
    base = dict(n_seq=2, n_draft=3, vocab=100, target_logits=0x1000, draft_ids=0x2000, uniforms=0x3000, tokens=0x4000,
                accepted=0x5000)
    return filled(_lib.VerifyArgs, "pcp_verify_args_init", **{**base, **kw})


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("fn,make,change,code,text", [
    ("pcp_top_logits", top, dict(n_rows=-1), -1, "n_rows"),
    ("pcp_top_logits", top, dict(n_rows=1 << 31), -1, "n_rows"),
    ("pcp_top_logits", top, dict(vocab=0), -1, "vocab"),
    ("pcp_top_logits", top, dict(vocab=(1 << 24) + 1), -1, "vocab"),
    ("pcp_top_logits", top, dict(k=0), -1, "k must"),
    ("pcp_top_logits", top, dict(k=257, vocab=1000), -1, "k must"),
    ("pcp_top_logits", top, dict(k=101), -1, "k must"),
    ("pcp_top_logits", top, dict(row_stride=99), -1, "row_stride"),
    ("pcp_top_logits", top, dict(row_stride=1 << 61), -9, "overflows"),
    ("pcp_top_logits", top, dict(logits_dtype=int(DType.f64)), -2, "logits dtype"),
    ("pcp_top_logits", top, dict(ids_dtype=int(DType.f32)), -2, "ids dtype"),
    ("pcp_top_logits", top, dict(temperature=0.0), -1, "temperature"),
    ("pcp_top_logits", top, dict(temperature=-1.0), -1, "temperature"),
    ("pcp_top_logits", top, dict(temperature=NAN), -1, "temperature"),
    ("pcp_top_logits", top, dict(temperature=INF), -1, "temperature"),
    ("pcp_top_logits", top, dict(temperature=1e-39), -1, "temperature"),
    ("pcp_top_logits", top, dict(flags=2), -1, "PCP_FLAG_ASYNC"),
    ("pcp_top_logits", top, dict(logits=None), -1, "NULL"),
    ("pcp_top_logits", top, dict(values=None), -1, "NULL"),
    ("pcp_top_logits", top, dict(ids=None), -1, "NULL"),
    ("pcp_top_logits", top, dict(logits=0x1001), -1, "element size"),
    ("pcp_top_logits", top, dict(ids=0x3004, ids_dtype=int(DType.i64)), -1, "element size"),
    ("pcp_top_logits", top, dict(lse=0x3002), -1, "element size"),
    ("pcp_top_logits", top, dict(), -1, "context is NULL"),
    ("pcp_distill_fwd_bwd", dist, dict(n_seq=0), -1, "n_seq"),
    ("pcp_distill_fwd_bwd", dist, dict(rows=-1), -1, "rows"),
    ("pcp_distill_fwd_bwd", dist, dict(vocab=0), -1, "vocab"),
    ("pcp_distill_fwd_bwd", dist, dict(vocab=(1 << 24) + 1), -1, "vocab"),
    ("pcp_distill_fwd_bwd", dist, dict(k=0), -1, "k must"),
    ("pcp_distill_fwd_bwd", dist, dict(k=257), -1, "k must"),
    ("pcp_distill_fwd_bwd", dist, dict(logit_seq_stride=3), -1, "logit_seq_stride"),
    ("pcp_distill_fwd_bwd", dist, dict(tok_offset=1), -1, "tok_offset"),
    ("pcp_distill_fwd_bwd", dist, dict(tok_offset=-1), -1, "tok_offset"),
    ("pcp_distill_fwd_bwd", dist, dict(tok_offset=(1 << 63) - 1), -1, "tok_offset"),
    ("pcp_distill_fwd_bwd", dist, dict(n_seq=1 << 30), -9, "rows"),
    ("pcp_distill_fwd_bwd", dist, dict(tok_seq_stride=1 << 61), -9, "token array"),
    ("pcp_distill_fwd_bwd", dist, dict(logits_dtype=int(DType.i32)), -2, "logits dtype"),
    ("pcp_distill_fwd_bwd", dist, dict(dlogits_dtype=int(DType.f16)), -2, "dlogits dtype"),
    ("pcp_distill_fwd_bwd", dist, dict(ids_dtype=int(DType.f32)), -2, "teacher_ids dtype"),
    ("pcp_distill_fwd_bwd", dist, dict(mask=0x6000, mask_dtype=int(DType.i64)), -2, "mask dtype"),
    ("pcp_distill_fwd_bwd", dist, dict(logits=None), -1, "NULL"),
    ("pcp_distill_fwd_bwd", dist, dict(teacher_ids=None), -1, "NULL"),
    ("pcp_distill_fwd_bwd", dist, dict(teacher_logits=None), -1, "NULL"),
    ("pcp_distill_fwd_bwd", dist, dict(logits=0x100001), -1, "element size"),
    ("pcp_distill_fwd_bwd", dist, dict(teacher_lse=0x6002), -1, "element size"),
    ("pcp_distill_fwd_bwd", dist, dict(dlogits=0x200002, dlogits_dtype=int(DType.f32)), -1, "element size"),
    ("pcp_distill_fwd_bwd", dist, dict(dlogits=0x100010), -1, "overlaps"),
    ("pcp_distill_fwd_bwd", dist, dict(dlogits=0x100000, dlogits_dtype=int(DType.f32)), -1, "overlaps"),
    ("pcp_distill_fwd_bwd", dist, dict(dlogits=0x100000), -1, "context is NULL"),
    ("pcp_distill_fwd_bwd", dist, dict(divergence=2), -1, "divergence"),
    ("pcp_distill_fwd_bwd", dist, dict(divergence=1), -1, "teacher_lse"),
    ("pcp_distill_fwd_bwd", dist, dict(temperature=0.0), -1, "temperature"),
    ("pcp_distill_fwd_bwd", dist, dict(temperature=NAN), -1, "temperature"),
    ("pcp_distill_fwd_bwd", dist, dict(weight=0.0), -1, "weight"),
    ("pcp_distill_fwd_bwd", dist, dict(weight=NAN), -1, "weight"),
    ("pcp_distill_fwd_bwd", dist, dict(loss_norm=-1.0), -1, "loss_norm"),
    ("pcp_distill_fwd_bwd", dist, dict(loss_norm=INF), -1, "loss_norm"),
    ("pcp_distill_fwd_bwd", dist, dict(flags=8), -1, "PCP_FLAG_ASYNC"),
    ("pcp_distill_fwd_bwd", dist, dict(), -1, "context is NULL"),
    ("pcp_verify_drafts", ver, dict(n_seq=-1), -1, "n_seq"),
    ("pcp_verify_drafts", ver, dict(n_seq=65536), -1, "n_seq"),
    ("pcp_verify_drafts", ver, dict(n_draft=-1), -1, "n_draft"),
    ("pcp_verify_drafts", ver, dict(n_draft=65), -1, "n_draft"),
    ("pcp_verify_drafts", ver, dict(vocab=0), -1, "vocab"),
    ("pcp_verify_drafts", ver, dict(vocab=(1 << 20) + 1), -1, "vocab"),
    ("pcp_verify_drafts", ver, dict(target_row_stride=99), -1, "strides"),
    ("pcp_verify_drafts", ver, dict(draft_row_stride=99), -1, "strides"),
    ("pcp_verify_drafts", ver, dict(target_row_stride=1 << 60), -9, "overflows"),
    ("pcp_verify_drafts", ver, dict(draft_row_stride=1 << 60), -9, "overflows"),
    ("pcp_verify_drafts", ver, dict(logits_dtype=int(DType.i32)), -2, "logits dtype"),
    ("pcp_verify_drafts", ver, dict(temperature=NAN), -1, "temperature"),
    ("pcp_verify_drafts", ver, dict(temperature=INF), -1, "temperature"),
    ("pcp_verify_drafts", ver, dict(uniforms=None), -1, "uniforms"),
    ("pcp_verify_drafts", ver, dict(uniforms=None, temperature=0.0), -1, "context is NULL"),
    ("pcp_verify_drafts", ver, dict(target_logits=None), -1, "NULL"),
    ("pcp_verify_drafts", ver, dict(tokens=None), -1, "NULL"),
    ("pcp_verify_drafts", ver, dict(accepted=None), -1, "NULL"),
    ("pcp_verify_drafts", ver, dict(draft_ids=None), -1, "draft_ids"),
    ("pcp_verify_drafts", ver, dict(draft_ids=None, n_draft=0), -1, "context is NULL"),
    ("pcp_verify_drafts", ver, dict(tokens=0x4004), -1, "element size"),
    ("pcp_verify_drafts", ver, dict(draft_logits=0x4001), -1, "element size"),
    ("pcp_verify_drafts", ver, dict(flags=4), -1, "PCP_FLAG_ASYNC"),
    ("pcp_verify_drafts", ver, dict(), -1, "context is NULL"),
])
def test_refusals(fn, make, change, code, text):
    L = _lib.lib()
    assert getattr(L, fn)(None, ctypes.byref(make(**change))) == code
    assert text in L.pcp_last_error(None).decode()


def test_null_args_and_defaults():
    L = _lib.lib()
    for fn in ("pcp_top_logits", "pcp_distill_fwd_bwd", "pcp_verify_drafts"):
        assert getattr(L, fn)(None, None) == -1 and "args is NULL" in L.pcp_last_error(None).decode()
    for fn in ("pcp_top_logits_args_init", "pcp_distill_args_init", "pcp_verify_args_init"):
        getattr(L, fn)(None)
    a = filled(_lib.DistillArgs, "pcp_distill_args_init")
    assert (a.logits_dtype, a.dlogits_dtype, a.ids_dtype, a.mask_dtype) == (DType.bf16, DType.bf16, DType.i32, DType.f32)
    assert a.temperature == 1.0 and a.weight == 1.0 and a.loss_norm == 0.0 and a.divergence == 0 and a.flags == 0
    t = filled(_lib.TopLogitsArgs, "pcp_top_logits_args_init")
    assert t.logits_dtype == DType.bf16 and t.ids_dtype == DType.i32 and t.temperature == 1.0
    v = filled(_lib.VerifyArgs, "pcp_verify_args_init")
    assert v.logits_dtype == DType.bf16 and v.temperature == 1.0 and v.flags == 0


def test_python_refusals():
    x = torch.zeros((2, 3, 50))
    ids, val, lse = torch.zeros((2, 3, 4), dtype=torch.int32), torch.zeros((2, 3, 4)), torch.zeros((2, 3))

    def refused(code, call):
        with pytest.raises(PcpError) as e:
            call()
        assert e.value.code == code

    refused(-1, lambda: distill.top_logits(x.transpose(1, 2), 3))
    refused(-1, lambda: distill.top_logits(x[:, ::2], 3))
    refused(-1, lambda: distill.distill_fwd_bwd(x[0], ids, val))
    refused(-1, lambda: distill.distill_fwd_bwd(x, ids[:, :2], val))
    refused(-1, lambda: distill.distill_fwd_bwd(x, ids, val[..., :3]))
    refused(-2, lambda: distill.distill_fwd_bwd(x, ids, val.double()))
    refused(-1, lambda: distill.distill_fwd_bwd(x, ids, val, lse[:1]))
    refused(-1, lambda: distill.distill_fwd_bwd(x, ids, val, lse, torch.ones(3, 3)))
    refused(-1, lambda: distill.distill_fwd_bwd(x, ids, val, lse, divergence="sideways"))
    d, u = torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 3))
    refused(-1, lambda: step.verify_drafts(x[0], d, uniforms=u))
    refused(-1, lambda: step.verify_drafts(x, d.int(), uniforms=u))
    refused(-1, lambda: step.verify_drafts(x, d[:, :1], uniforms=u))
    refused(-1, lambda: step.verify_drafts(x, d, x, uniforms=u))
    refused(-1, lambda: step.verify_drafts(x, d, x[:, :2].bfloat16(), uniforms=u))
    refused(-1, lambda: step.verify_drafts(x, d, uniforms=u[:, :2]))
    refused(-1, lambda: step.verify_drafts(x, d, uniforms=u.double()))
    refused(-1, lambda: step.verify_drafts(x, d, uniforms=u, draft_lens=torch.zeros(2, dtype=torch.int64)))


@pytest.mark.parametrize("forward,tail", [(True, True), (True, False), (False, True)])
def test_reference_gradient_against_differences(forward, tail):
    rng = np.random.default_rng(0)
    V, h = 30, 1e-6
    x, t = rng.standard_normal(V) * 2, rng.standard_normal(4) * 2
    ids = np.array([3, 7, -100, 9])
    full = rng.standard_normal(V)
    full[[3, 7, 9]] = t[[0, 1, 3]]
    lse = float(lse_ref(full[None])[0]) if tail else None

    def loss(z):
        return row_ref(z, ids, t, lse, 1.3, forward)[0]

    g = row_ref(x, ids, t, lse, 1.3, forward)[1] / 1.3
    num = np.array([(loss(x + h * e) - loss(x - h * e)) / (2 * h) for e in np.eye(V)])
    assert np.abs(num - g).max() < 1e-8


def test_references_on_small_rows():
    v, i, lse = top_ref(np.array([[1.0, 3.0, 3.0, -np.inf]]), 3)
    assert i.tolist() == [[1, 2, 0]] and v.tolist() == [[3.0, 3.0, 1.0]]
    assert abs(lse[0] - np.log(np.e + 2 * np.e ** 3)) < 1e-12
    x = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.8, 0.1]]]))
    y = np.log(np.array([[[0.2, 0.6, 0.2]]]))
    for u0, want in ((0.4, ([1, 1], 1)), (0.6, ([0, -100], 0))):   # p/q of token 1 is 0.5
        tok, acc, _ = verify_ref(x, y, np.array([[1]]), [1], np.array([[u0, 0.5]]), 1.0, 3)
        assert tok[0].tolist() == want[0] and acc[0] == want[1]


def test_rows_that_overlap_are_refused():
    """Expanded rows lie 0 elements apart, which the C entry takes for "vocab apart"."""
    import torch

    from pcp_amd import distill, step
    from pcp_amd._lib import PcpError
    with pytest.raises(PcpError, match="overlap"):
        distill.top_logits(torch.zeros(1, 16).expand(4, 16), 2)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(PcpError, match="overlap"):
        step.verify_drafts(torch.zeros(1, 1, 16).expand(2, 4, 16), ids, temperature=0.0)
    with pytest.raises(PcpError, match="overlap"):
        step.verify_drafts(torch.zeros(2, 4, 16), ids, torch.zeros(1, 1, 16).expand(2, 3, 16))
    with pytest.raises(PcpError, match="overlap"):
        step.verify_drafts(torch.zeros(1, 1, 16).expand(2, 1, 16), ids[:, :0], temperature=0.0)
    assert step._row_stride(torch.zeros(2, 4, 16)[:, :, :10]) == 16
    assert step._row_stride(torch.zeros(2, 0, 16)) == 16
