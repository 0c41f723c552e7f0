"""Gradient norm, clipping and the update of many tensors on the GPU.

The norm is summed in f64 and rounded to f32 once, the coefficient is f64's quotient rounded once: 2^-24 of
themselves each (and 2^-40 for the f64 sum of up to 2^28 squares, far below). From the device's own
coefficient on everything is one f32 rounding per operation, in a stated order: bits are compared.
"""
import numpy as np
import pytest
import torch

from pcp_amd import grpo, step
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
STEP = 2.0 ** -24 * (1 + 1e-6)

LISTS = [
    [(5, F32)], [(1, BF16)], [(0, F32), (3, F16), (0, BF16), (1, F32)], [(16384, F32), (16385, BF16), (16383, F16)],
    [(4096 + i, (F32, BF16, F16)[i % 3]) for i in range(7)], [(i % 11, (F16, F32, BF16)[i % 3]) for i in range(700)],
    [(3_000_001, BF16), (1_000_003, F32), (77, F16)], [(20_000_000, F32)], [(1000, F32)] * 241, [(900, BF16)] * 161,
]


def tensors(sizes, seed=0, scale=1e-2, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for n, t in sizes:
        buf = torch.empty(n + offset, dtype=t, device=DEV)
        v = buf[offset:]
        v.copy_(torch.randn(n, generator=g, device=DEV) * scale)
        out.append(v)
    return out


def norm_of(grads, kind):
    flat = np.concatenate([g.double().cpu().numpy() for g in grads])
    return (np.sqrt((flat * flat).sum()) if kind == "l2" else np.abs(flat).max(initial=0.0))


def check_norm(got, grads, kind, max_norm):
    want = norm_of(grads, kind)
    assert abs(float(got.norm) - want) <= STEP * want
    coef = min(1.0, max_norm / want) if want else 1.0
    assert abs(float(got.coef) - coef) <= STEP * coef


@pytest.mark.parametrize("sizes", LISTS, ids=range(len(LISTS)))
@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_and_clip(sizes, kind, offset):
    grads = tensors(sizes, 1, offset=offset)
    want = norm_of(grads, kind)
    check_norm(step.grad_norm(grads, norm_type=kind), grads, kind, float("inf"))
    for most in (0.3 * want, 2 * want):
        most = float(np.float32(most))
        before = [g.clone() for g in grads]
        got = step.clip_grads(grads, most, norm_type=kind)
        check_norm(got, before, kind, most)
        for a, b in zip(grads, before):
            assert torch.equal(a, (b.float() * got.coef).to(b.dtype))


@pytest.mark.parametrize("to", [F32, BF16, F16])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_clip_into_other_types(to, offset):
    sizes = LISTS[4] + LISTS[5] + [(100_001, F32), (70_001, BF16)]
    grads = tensors(sizes, 2, offset=offset, scale=0.5)
    before = [g.clone() for g in grads]
    total = sum(n for n, _ in sizes)
    flat = torch.full((total + 8,), 3.0, dtype=to, device=DEV)
    out = list(flat[offset:offset + total].split([n for n, _ in sizes]))
    got = step.clip_grads(grads, 1.0, out=out)
    check_norm(got, before, "l2", 1.0)
    for a, b, o in zip(grads, before, out):
        assert torch.equal(a, b) and torch.equal(o, (b.float() * got.coef).to(to))
    assert (flat[:offset] == 3).all() and (flat[offset + total:] == 3).all()


def test_sizes_of_values():
    """Squares that leave f32's range, subnormal gradients, all zeros, nothing at all."""
    for v in (1e30, 1e-30, 1e-42):
        g = torch.full((1000,), v, device=DEV)
        want = float(g[0].double()) * np.sqrt(1000)
        n = step.grad_norm(g)
        assert abs(float(n.norm) - want) <= max(STEP * want, 2.0 ** -150)
        got = step.clip_grads(g, want / 2 if v > 1e-40 else 1.0)
        assert float(got.coef) == (1.0 if v <= 1e-40 else pytest.approx(0.5, rel=1e-6))
    z = torch.zeros(100, device=DEV)
    assert float(step.clip_grads(z, 1.0).coef) == 1.0 and float(step.grad_norm([z, z]).norm) == 0.0
    got = step.grad_norm([torch.zeros(0, device=DEV)], 1.0)
    assert float(got.norm) == 0.0 and float(got.coef) == 1.0
    got = step.grad_norm([], 1.0, ctx=grpo.default_context(0))
    assert float(got.norm) == 0.0 and float(got.coef) == 1.0


@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite(kind, bad):
    """Reported; gradients, parameters and velocities stay as they are."""
    grads = tensors([(5000, F32), (333, BF16), (70, F16)], 3)
    grads[1][7] = bad
    before = [g.clone() for g in grads]
    ctx = grpo.Context(0)
    got = step.clip_grads(grads, 1e-3, norm_type=kind, sync=False, ctx=ctx)
    p, v = tensors([(5000, F32), (333, F32), (70, F32)], 4), tensors([(5000, F32), (333, F32), (70, F32)], 5)
    b = [torch.ones(t.numel(), dtype=BF16, device=DEV) for t in p]
    had = [t.clone() for t in p + v + b]
    step.nesterov_update_many(p, v, grads, b, coef=got.coef, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -4 and torch.isnan(got.coef) and not torch.isfinite(got.norm)
    for a, c in zip(grads, before):
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))
    for a, c in zip(p + v + b, had):
        assert torch.equal(a, c)
    grads[1][7] = 0
    assert np.isfinite(float(step.clip_grads(grads, 1.0, ctx=ctx).coef))


def plain_update(p, v, g, coef, lr, mu, mode):
    """On the CPU in f32, one rounding per operation."""
    lr, mu, g = np.float32(lr), np.float32(mu), np.float32(coef) * g
    if mode == "sutskever":
        v = mu * v + g
        return p - lr * (g + mu * v), v
    v = mu * v + lr * g
    return p - v, v


@pytest.mark.parametrize("sizes", LISTS, ids=range(len(LISTS)))
@pytest.mark.parametrize("mode", ["sutskever", "mlir"])
@pytest.mark.parametrize("offset,copies", [(0, "all"), (1, "some"), (0, "none"), (3, "all")])
def test_update_many(sizes, mode, offset, copies):
    grads = tensors(sizes, 6, offset=offset)
    counts = [n for n, _ in sizes]
    total = sum(counts)
    flat_p, flat_v = (torch.randn(total + 8, device=DEV) for _ in range(2))
    flat_b = torch.full((total + 8,), 9.0, dtype=BF16, device=DEV)
    had_p, had_v = flat_p.cpu().numpy(), flat_v.cpu().numpy()
    p, v, b = ([*t[o:o + total].split(counts)] for t, o in ((flat_p, offset), (flat_v, 2 - offset % 2), (flat_b, offset)))
    if copies == "some":
        b = [x if i % 2 else None for i, x in enumerate(b)]
    coef = torch.tensor(0.37, device=DEV) if copies != "none" else None
    c = np.float32(0.37) if coef is not None else np.float32(1)
    step.nesterov_update_many(p, v, grads, None if copies == "none" else b, coef=coef, learning_rate=0.03, momentum=0.85, mode=mode)
    at = 0
    new_p, new_v = flat_p.cpu().numpy(), flat_v.cpu().numpy()
    vo = 2 - offset % 2
    for n, g in zip(counts, grads):
        want_p, want_v = plain_update(had_p[offset + at:offset + at + n], had_v[vo + at:vo + at + n], g.float().cpu().numpy(), c,
                                      0.03, 0.85, mode)
        assert np.array_equal(new_p[offset + at:offset + at + n], want_p) and np.array_equal(new_v[vo + at:vo + at + n], want_v)
        at += n
    for new, had, o in ((new_p, had_p, offset), (new_v, had_v, vo)):
        assert np.array_equal(new[:o], had[:o]) and np.array_equal(new[o + total:], had[o + total:])
    want_b = torch.full_like(flat_b, 9.0)
    for i, (w, new) in enumerate(zip(want_b[offset:offset + total].split(counts), p)):
        if copies == "all" or (copies == "some" and i % 2):
            w.copy_(new)
    assert torch.equal(flat_b, want_b)


def test_an_optimizers_own_velocities():
    """update_many and update_flat of one optimizer give the same bits, and its state serializes alike."""
    counts = [1000, 0, 77, 4096]
    total = sum(counts)
    a, b = step.Nesterov(counts, 0.02, 0.8), step.Nesterov(counts, 0.02, 0.8)
    p = torch.randn(total, device=DEV)
    q = p.clone()
    for i in range(3):
        g = torch.randn(total, device=DEV)
        s1, s2 = (torch.empty(total, dtype=BF16, device=DEV) for _ in range(2))
        a.update_flat(p, g, s1)
        b.update_many(q.split(counts), g.split(counts), s2.split(counts))
        assert torch.equal(p, q) and torch.equal(s1, s2)
    assert a.serialize() == b.serialize()
    with pytest.raises(PcpError):
        b.update_many(q.split([1000, 77, 4096]), g.split([1000, 77, 4096]))


def test_refusals_on_the_device():
    g = torch.randn(10, device=DEV)
    for call in (lambda: step.clip_grads([g, g], 1.0), lambda: step.clip_grads([g], 1.0, out=[g[:9]]),
                 lambda: step.clip_grads([g], 0.0), lambda: step.clip_grads([g.double()], 1.0),
                 lambda: step.clip_grads([g.view(2, 5).t()], 1.0), lambda: step.grad_norm([g.cpu()]),
                 lambda: step.nesterov_update_many([g], [g.clone()], [torch.randn(11, device=DEV)]),
                 lambda: step.nesterov_update_many([g], [g], [g.clone()]),
                 lambda: step.nesterov_update_many([g.to(BF16)], [g], [g.clone()]),
                 lambda: step.nesterov_update_many([g], [g.clone()], [g.clone()], coef=g[:2])):
        before = g.clone()
        with pytest.raises(PcpError):
            call()
        assert torch.equal(g, before)
    n = step.grad_norm([g, g])          # without outputs a gradient may stand there twice
    assert abs(float(n.norm) - np.sqrt(2) * norm_of([g], "l2")) < 1e-5


def test_captured_and_on_other_streams():
    """Norm, clipping and update in one graph, replayed on new gradients; the coefficient never visits the host."""
    sizes = LISTS[4]
    counts = [n for n, _ in sizes]
    grads = tensors(sizes, 7)
    p, v = (list(torch.randn(sum(counts), device=DEV).split(counts)) for _ in range(2))
    b = list(torch.zeros(sum(counts), dtype=BF16, device=DEV).split(counts))
    clipped = [torch.empty(n, device=DEV) for n in counts]
    ctx = grpo.Context(0)
    out = step.clip_grads(grads, 0.5, out=clipped, ctx=ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.clip_grads(grads, 0.5, out=clipped, outputs=out, sync=False, ctx=ctx)
        step.nesterov_update_many(p, v, grads, b, coef=out.coef, sync=False, ctx=ctx)
    for turn in range(4):
        for g in grads:
            g.copy_(torch.randn(g.numel(), device=DEV) * 10.0 ** (turn - 3))
        ep, ev = [x.clone() for x in p], [x.clone() for x in v]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step.grad_norm(grads, 0.5)
        assert torch.equal(out.norm, want.norm) and torch.equal(out.coef, want.coef)
        step.nesterov_update_many(ep, ev, grads, coef=want.coef)
        for a, c in zip(p + v, ep + ev):
            assert torch.equal(a, c)
        for g, c in zip(grads, clipped):
            assert torch.equal(c, g.float() * want.coef)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = step.clip_grads(grads, 0.5, out=clipped, stream=st)
    assert torch.equal(got.norm, want.norm)


def test_a_tensor_of_several_pieces():
    """More than 2^28 elements in one tensor: pieces of it, and 64-bit places."""
    n = (1 << 28) + 12345
    g = torch.zeros(n, dtype=BF16, device=DEV)
    g[-3:] = 2.0
    g[1 << 28] = 1.0
    got = step.clip_grads(g, 1.0, out=torch.empty(n, dtype=BF16, device=DEV))
    assert abs(float(got.norm) - np.sqrt(13)) <= STEP * np.sqrt(13)
    p, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    step.nesterov_update_many([p], [v], [g], learning_rate=1.0, momentum=0.0)
    assert torch.equal(p, -g.float()) and torch.equal(v, g.float())
