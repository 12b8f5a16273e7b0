"""Norms over many gradients and clipping against float64.

Tolerance: squares and sums are double, so a norm is off by its rounding to float32, 2^-24, and the double sum's few units of
2^-53; a scaled gradient by the factor's rounding (2^-24), the product's (2^-24) and the type's (bf16 2^-8)."""

import math

import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gc():
    return load_package().grad_clip


def make(shapes, dtypes=(BF16,), std=1e-2, seed=0):
    print(f"[case] {shapes[:6]} .. {len(shapes)}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(*s, generator=g, device=DEV) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def exact_norms(grads, per_adapter):
    n = grads[0].shape[0] if per_adapter else 1
    return sum(g.double().reshape(n, -1).square().sum(1) for g in grads).sqrt()


def check(gc, grads, limits, per_adapter):
    norms = exact_norms(grads, per_adapter)
    out, got = gc.clip_grad_norm(grads, limits, per_adapter=per_adapter)
    assert got.shape == ((len(norms),) if per_adapter else ())
    assert bool(((got.double() - norms).abs() <= norms * 2.0 ** -23).all())
    assert torch.equal(got, gc.grad_norm(grads, per_adapter=per_adapter))
    lim = torch.as_tensor(limits, dtype=torch.float64, device=DEV).expand(len(norms))
    factor = torch.where(norms > lim, lim / norms, 1.0)
    for g, o in zip(grads, out):
        f = factor.view(-1, *[1] * (g.ndim - 1)) if per_adapter else factor[0]
        want = g.double() * f
        tol = want.abs() * ((2.0 ** -8 if g.dtype == BF16 else 2.0 ** -24) + 2.0 ** -22) + (torch.finfo(g.dtype).smallest_normal * 2.0 ** -7)
        assert o.dtype == g.dtype and bool(((o.double() - want).abs() <= tol).all())
        for a in range(len(norms)):  # unclipped gradients keep their bits
            if per_adapter and norms[a] < lim[a] * 0.999:
                assert torch.equal(o[a], g[a])
    mine = [g.clone() for g in grads]
    assert torch.equal(gc.clip_grad_norm_(mine, limits, per_adapter=per_adapter), got)
    assert all(torch.equal(a, b) for a, b in zip(mine, out))


@pytest.mark.parametrize("shapes,dtypes", [
    ([(1,)], (BF16,)), ([(3,), (5,)], (F32,)), ([(7, 9), (33,), (1, 1, 1), (1000,)], (BF16, F32)),
    ([(4096, 16), (16, 1024)] * 3, (BF16,)), ([(32769,), (32767,), (65536,), (131073,)], (BF16, F32)), ([(5, 3)] * 500, (F32, BF16)),
    ([(3000001,)], (F32,))])
def test_one_norm(gc, shapes, dtypes):
    grads = make(shapes, dtypes)
    norm = float(exact_norms(grads, False))
    for limit in (norm * 0.3, norm * 2, 0.0):
        check(gc, grads, limit, False)


@pytest.mark.parametrize("n_ad,shapes,dtypes", [
    (1, [(64, 8), (8, 24)], (BF16,)), (2, [(7, 3), (3, 5)], (F32,)), (4, [(4096, 16), (16, 1024)] * 7, (BF16,)),
    (5, [(33, 7), (7, 91), (1,)], (BF16, F32)), (8, [(3, 11)] * 130, (BF16,)), (3, [(70001,), (13,)], (BF16, F32))])
def test_norms_of_adapters(gc, n_ad, shapes, dtypes):
    grads = make([(n_ad, *s) for s in shapes], dtypes, seed=1)
    norms = exact_norms(grads, True)
    limits = (norms * torch.where(torch.arange(n_ad, device=DEV) % 2 == 0, 0.4, 2.5)).float()
    check(gc, grads, limits, True)
    check(gc, grads, float(norms.mean()) * 0.7, True)


def test_squares_beyond_float32(gc):
    big = [torch.full((8,), 2.0 ** 100, device=DEV), torch.full((8,), 2.0 ** 100, device=DEV)]
    out, norm = gc.clip_grad_norm(big, 4.0)
    assert float(norm) == 2.0 ** 102 and all(torch.equal(o, torch.ones(8, device=DEV)) for o in out)
    small = [torch.full((4,), 2.0 ** -120, device=DEV)]
    assert float(gc.grad_norm(small)) == 2.0 ** -119


def test_what_is_not_finite_stays_in_its_adapter(gc):
    grads = make([(4, 30), (4, 9, 5)])
    want, _ = gc.clip_grad_norm(grads, 1e-3, per_adapter=True)
    grads[0][1, 3], grads[1][2, 0, 0] = float("nan"), float("inf")
    out, norms = gc.clip_grad_norm(grads, 1e-3, per_adapter=True)
    assert math.isnan(norms[1]) and math.isinf(norms[2]) and torch.isfinite(norms[[0, 3]]).all()
    for o, w, g in zip(out, want, grads):
        assert torch.equal(o[[0, 3]], w[[0, 3]])
        assert torch.equal(o[1].view(torch.int16), g[1].view(torch.int16))  # no factor can be had: as they are
    assert int(torch.isnan(out[1][2]).sum()) == 1 and int(out[1][2].nonzero().shape[0]) == 1  # all but the infinity become zero
    limits = torch.tensor([float("nan"), -1.0, 1e-3, 1e9], device=DEV)
    fine = make([(4, 30)])
    out, _ = gc.clip_grad_norm(fine, limits, per_adapter=True)
    assert torch.equal(out[0][0], fine[0][0]) and not out[0][1].any() and torch.equal(out[0][3], fine[0][3])


def test_empty_tensors_and_odd_places(gc):
    grads = make([(3, 10), (3, 0), (3, 4)])
    check(gc, grads, 0.01, True)
    assert not gc.grad_norm([torch.empty(2, 0, device=DEV)], per_adapter=True).any()
    flat = make([(3 * 1001 + 5,)])[0]
    views = [flat[1:1 + 3 * 500].view(3, 500), flat[1502:1502 + 3 * 333].view(3, 333)]  # 2 and 12 bytes past 16
    out = torch.zeros(4000, dtype=BF16, device=DEV)
    outs = [out[3:1503].view(3, 500), out[1600:1600 + 999].view(3, 333)]
    limits = torch.tensor([1e-3, 1e9, 1e-2], device=DEV)
    want, norms = gc.clip_grad_norm([v.clone() for v in views], limits, per_adapter=True)
    got, n = gc.GradClipPlan(views, limits, per_adapter=True, out=outs).run()
    assert torch.equal(n, norms) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert not out[:3].any() and not out[1503:1600].any() and not out[2599:].any()


def test_plan_reads_its_buffers_at_every_run_and_replays(gc):
    shapes = [(4, 100, 8), (4, 8, 333)] * 70  # two launches of either kernel
    grads = make(shapes)
    limits = torch.full((4,), 0.05, device=DEV)
    plan = gc.GradClipPlan(grads, limits, per_adapter=True)
    graph = torch.cuda.CUDAGraph()
    plan.run()
    with torch.cuda.graph(graph):
        out, norms = plan.run()
    for step in range(3):
        for g, f in zip(grads, make(shapes, seed=step + 10)):
            g.copy_(f)
        limits.fill_(0.02 * (step + 1))
        graph.replay()
        want, wn = gc.clip_grad_norm(grads, limits, per_adapter=True)
        torch.cuda.synchronize()
        assert torch.equal(norms, wn) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_gradient_given_twice(gc):
    grad = torch.ones(4, 8, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        gc.clip_grad_norm_([grad, grad], 1.0)
    with pytest.raises(ValueError, match="twice|overlap"):
        gc.clip_grad_norm_([grad, grad[0]], 1.0)
    (one, two), norm = gc.clip_grad_norm([grad, grad], 4.0)
    assert float(norm) == 8.0 and torch.equal(one, two) and one.data_ptr() != two.data_ptr() and float(one[0, 0]) == 0.5
    assert float(gc.grad_norm([grad, grad])) == 8.0


def test_a_tensor_beyond_32_bits(gc):
    """2^31 + 8 ones: the norm's square is exact in float64, the scaled values are powers of two."""
    n = (1 << 31) + 8
    grad = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    grad[-8:] = 0
    norm = gc.clip_grad_norm_([grad], (2.0 ** 31) ** 0.5 / 4)
    assert abs(float(norm) - (2.0 ** 31) ** 0.5) <= (2.0 ** 31) ** 0.5 * 2.0 ** -24
    assert torch.equal(grad[:1000], torch.full((1000,), 0.25, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(grad[-1008:-8], torch.full((1000,), 0.25, dtype=torch.bfloat16, device=DEV)) and not grad[-8:].any()


def test_two_plans_at_once(gc):
    g = torch.Generator(device=DEV).manual_seed(11)
    sets = [[torch.randn(2, c, generator=g, device=DEV) for c in (100000, 77, 300001)] for _ in range(2)]
    want = [gc.clip_grad_norm(s, 1.0, per_adapter=True) for s in sets]
    plans = [gc.GradClipPlan(s, 1.0, per_adapter=True) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for plan, stream in zip(plans, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                plan.run()
    torch.cuda.synchronize()
    for plan, (out, norms) in zip(plans, want):
        assert torch.equal(plan.norms, norms) and all(torch.equal(a, b) for a, b in zip(plan.out, out))


@pytest.mark.parametrize("n", [120, 121, 240, 1000, 4500])
def test_many_tensors(gc, n):
    """More tensors than a launch's arguments hold, empty ones among them, from plans that run again, in a captured graph too."""
    g = torch.Generator(device=DEV).manual_seed(n)
    sizes = [(7 * i) % 61 if i % 9 else 0 for i in range(n)]
    sizes[n // 2] = 70001
    grads = [torch.randn(2, s, generator=g, device=DEV).to(torch.bfloat16 if i % 3 else torch.float32) for i, s in enumerate(sizes)]
    limits = torch.tensor([3.0, 1e6], device=DEV)

    def check(out, norms):
        want = torch.stack([t.double().square().sum(1) for t in grads]).sum(0).sqrt()
        assert bool(((norms.double() - want).abs() <= 2.0 ** -23 * want).all())
        for t, o in zip(grads, out):
            scaled = t[0].double() * (3.0 / want[0])
            step = 2.0 ** -8 if t.dtype == torch.bfloat16 else 2.0 ** -24
            assert bool(((o[0].double() - scaled).abs() <= (step + 2.0 ** -22) * scaled.abs() + 1e-40).all()) and torch.equal(o[1], t[1])

    check(*gc.clip_grad_norm(grads, limits, per_adapter=True))
    captured, eager = (gc.GradClipPlan(grads, limits, per_adapter=True) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # (a plan whose first run is captured)
        captured.run()
    for turn in range(3):
        for t in grads:
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        check(*eager.run())
        graph.replay()
        check(captured.out, captured.norms)
        if turn == 1:
            check(*captured.run())
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):  # (and one that has run before)
        eager.run()
    for t in grads:
        t.mul_(0.5)
    again.replay()
    check(eager.out, eager.norms)


@pytest.mark.parametrize("native", [True, False])
def test_tables_of_the_host_module_and_of_python(gc, monkeypatch, native):
    """What both ways of making a table take and refuse, and that they give the same bits."""
    want, norms = gc.clip_grad_norm([torch.arange(12, device=DEV).float().view(2, 6), torch.ones(2, 3, device=DEV).to(torch.bfloat16)], 2.0, per_adapter=True)
    if not native:
        monkeypatch.setattr(load_package()._native, "host", lambda: None)
    grads = [torch.nn.Parameter(torch.arange(12, device=DEV).float().view(2, 6)), torch.ones(2, 3, device=DEV).to(torch.bfloat16), torch.empty(2, 0, device=DEV)]
    bucket = torch.empty(12 * 4 + 6 * 2, dtype=torch.uint8, device=DEV)
    outs = [bucket[:48].view(torch.float32).view(2, 6), bucket[48:].view(torch.bfloat16).view(2, 3), torch.empty(2, 0, device=DEV)]
    out, got = gc.GradClipPlan(grads, 2.0, per_adapter=True, out=outs).run()
    assert torch.equal(got, norms) and all(torch.equal(a, b) for a, b in zip(out, want))
    f = torch.zeros(40, device=DEV)
    plan = lambda g, o, per=False: gc.GradClipPlan(g, 1.0, per_adapter=per, out=o)
    plan([f[:10], f[10:20]], [f[:10], f[10:20]])        # in place
    plan([f[:10], f[:10]], [f[20:30], f[30:]])          # one gradient read twice
    plan([f[:10], f[5:15]], [f[20:30], f[30:]])
    for g, o in (([f[:10], f[5:15]], [f[:10], f[20:30]]), ([f[:10], f[10:20]], [f[10:20], f[20:30]]), ([f[:10], f[20:30]], [f[30:], f[25:35]]),
                 ([f[:20]], [f[10:30]]), ([f[10:30]], [f[:20]]), ([f[5:6], f[:10]], [f[20:21], f[:10]]), ([f[:10], f[5:6]], [f[:10], f[20:21]])):
        with pytest.raises(ValueError, match="overlap"):
            plan(g, o)
    for g, o, message in (([f[:10]], [f[20:31]], "out must be"), ([f[:10]], [f[20:30].to(torch.bfloat16)], "out must be"), ([f[:10]], [], "names 0"),
                          ([f[::2]], None, "contiguous"), ([f[:10]], [f[20:40:2]], "out must be")):
        with pytest.raises(ValueError, match=message):
            plan(g, o)
    with pytest.raises(ValueError, match="leading axis"):
        plan([torch.zeros(2, 3, device=DEV), torch.zeros(3, 2, device=DEV)], None, True)
    with pytest.raises(ValueError, match="1 to 65535"):
        plan([torch.zeros(0, 3, device=DEV)], None, True)
    with pytest.raises(TypeError, match="BF16"):
        plan([f, f.double()], None)
    with pytest.raises(RuntimeError, match="GPU"):
        plan([f, f.cpu()], None)
