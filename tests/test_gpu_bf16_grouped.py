"""Products grouped by expert on bf16 weights and their gradients against float64.

Tolerance: products of bf16 values are exact in float32, so a sum of d of them is off by at most d * 2^-23 * S (S the sum of the
products' magnitudes; one unit of the last place an addition, whichever way the matrix instruction rounds), and the one
rounding to bf16 by half a step, 2^-8 of the value."""

import numpy
import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def gl():
    return load_package().bf16_grouped_linear


def make(rows, k, n, sizes, seed=0):
    print(f"[case] {rows} rows, {k} -> {n}, sizes {sizes if len(sizes) < 20 else len(sizes)}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    return t(rows, k), t(len(sizes), k, n), t(rows, n), torch.tensor(sizes, dtype=torch.int32, device=DEV)


def spans(rows, sizes):
    at = 0
    for g, s in enumerate(sizes):
        s = min(max(0, s), rows)
        yield g, slice(min(at, rows), min(at + s, rows))
        at += s


def exact_forward(x, w, sizes):
    out = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    for g, r in spans(x.shape[0], sizes):
        out[r] = x[r].double() @ w[g].double()
    return out


def exact_dw(x, dy, sizes):
    out = torch.zeros(len(sizes), x.shape[1], dy.shape[1], dtype=torch.float64, device=x.device)
    for g, r in spans(x.shape[0], sizes):
        out[g] = x[r].double().T @ dy[r].double()
    return out


def close(got, want, magnitudes, depth):
    tol = depth * 2.0 ** -23 * magnitudes + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0.0)
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(got).any() and float(off.max()) <= 0.0, f"{float(off.max())} beyond at {int(off.argmax())}"


def check(gl, x, w, dy, sizes_t, sizes, dw_dtype=torch.bfloat16, flags=0):
    k, n = w.shape[1:]
    close(gl.grouped_matmul(x, w, sizes_t, flags=flags), exact_forward(x, w, sizes), exact_forward(x.abs(), w.abs(), sizes), k)
    dx, dw = gl.grouped_matmul_backward(x, dy, w, sizes_t, dw_dtype=dw_dtype, flags=flags)
    wt = w.transpose(1, 2)
    close(dx, exact_forward(dy, wt, sizes), exact_forward(dy.abs(), wt.abs(), sizes), n)
    assert dw.dtype == dw_dtype
    close(dw, exact_dw(x, dy, sizes), exact_dw(x.abs(), dy.abs(), sizes), max(1, max(min(max(0, s), x.shape[0]) for s in sizes)))


@pytest.mark.parametrize("rows,k,n,sizes", [
    (1, 8, 8, [1]),                                   # the least
    (1, 64, 128, [0, 0, 1, 0]),
    (5, 72, 40, [0, 2, 0, 3, 0]),                     # nothing is a multiple of a tile
    (64, 512, 768, [1] * 64),                         # decode: a row a group
    (127, 136, 264, [127]),
    (129, 128, 128, [0, 129]),
    (300, 200, 328, [3, 128, 0, 129, 40]),
    (1003, 712, 1096, [100, 0, 250, 1, 7, 0, 0, 333, 64, 65, 63, 20, 81]),  # rows behind the last group
    (1537, 264, 520, [17] * 60 + [500]),
    (2048, 1024, 512, [2048]),
    (2000, 512, 1024, [900, 700, 400]),
    (700, 64, 64, [1] * 500 + [0] * 523 + [200]),     # as many groups as there may be
])
def test_against_float64(gl, rows, k, n, sizes):
    x, w, dy, st = make(rows, k, n, sizes)
    check(gl, x, w, dy, st, sizes)
    check(gl, x, w, dy, st, sizes, torch.float32)


@pytest.mark.parametrize("tile", ["256X256", "128X256", "64X128"])
@pytest.mark.parametrize("rows,k,n,sizes", [
    (1, 8, 8, [1]), (70, 200, 72, [0, 30, 5, 0, 35]), (257, 64, 264, [257]), (900, 328, 520, [3, 300, 0, 129, 40, 64, 65, 200]),
    (3000, 136, 1000, [100, 900, 0, 1, 255, 256, 257, 700, 17, 300, 40, 60]),  # several tiles a workgroup
    (2500, 1032, 2056, [7, 0, 1500, 600, 64, 128, 100]), (1100, 2056, 1544, [1] * 100 + [0] * 20 + [500, 400])])
def test_each_tile(gl, rows, k, n, sizes, tile):
    flags = getattr(load_package()._native, f"FLAG_BF16_GROUPED_TILE_{tile}")
    x, w, dy, st = make(rows, k, n, sizes, seed=1)
    check(gl, x, w, dy, st, sizes, flags=flags)
    check(gl, x, w, dy, st, sizes, torch.float32, flags=flags)
    for dtype in (torch.bfloat16, torch.float32):  # in one launch and by themselves: the same bits
        dx, dw = gl.grouped_matmul_backward(x, dy, w, st, dw_dtype=dtype, flags=flags)
        assert torch.equal(dx, gl.grouped_matmul_backward(None, dy, w, st, need_dw=False, flags=flags)[0])
        assert torch.equal(dw, gl.grouped_matmul_backward(x, dy, None, st, need_dx=False, dw_dtype=dtype, flags=flags)[1])


@pytest.mark.parametrize("rows,k,n,groups", [
    (4051, 128, 120, 22), (886, 168, 736, 13), (1003, 712, 1096, 13), (4096, 1024, 1024, 8), (300, 64, 280, 28), (8000, 1576, 1744, 25), (1, 8, 8, 1), (70, 40, 136, 1024)])
def test_both_gradients_and_each(gl, rows, k, n, groups):
    """The sizes at which both come from one launch, with empty and uneven groups and spare rows, against float64 and in a captured graph."""
    g = torch.Generator().manual_seed(rows)
    share = torch.rand(groups, generator=g) ** 2 * (torch.rand(groups, generator=g) > 0.25)
    share[0] += 0.01
    sizes = (share / share.sum() * rows * 0.97).long().tolist()
    x, w, dy, st = make(rows, k, n, sizes, seed=6)
    check(gl, x, w, dy, st, sizes)
    check(gl, x, w, dy, st, sizes, torch.float32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, dw = gl.grouped_matmul_backward(x, dy, w, st)
    for turn in range(3):
        dy.copy_(torch.randn(dy.shape, device=DEV))
        st.copy_(st.roll(1))
        graph.replay()
        got = dx.clone(), dw.clone()
        assert all(torch.equal(a, b) for a, b in zip(got, gl.grouped_matmul_backward(x, dy, w, st))), turn


@pytest.mark.parametrize("sizes", [[0, 0, 0], [40, 200, 7], [-5, 40, -1], [1 << 30, 5, 1 << 30], [100, 0, 0]])
def test_sizes_that_do_not_fit_the_rows(gl, sizes):
    x, w, dy, st = make(100, 96, 72, sizes)
    check(gl, x, w, dy, st, sizes)


def test_longest_depths(gl):
    for rows, k, n in ((70, 16384, 64), (40, 64, 24576), (9000, 64, 96)):
        sizes = [rows // 2, rows - rows // 2]
        x, w, dy, st = make(rows, k, n, sizes)
        check(gl, x, w, dy, st, sizes, torch.float32)


@pytest.mark.parametrize("rows,k,n,sizes,parts", [
    (1, 4096, 512, [0, 1, 0], "f"), (1, 512, 4104, [1], "d"), (8, 704, 8952, [0, 2, 1, 0, 5, 0], "d"), (70, 4168, 72, [9, 0, 30, 1, 20], "f"),
    (200, 72, 4232, [9, 0, 130, 1, 20], "d"), (9000, 8, 520, [9000], "w"), (9100, 264, 40, [5000, 0, 4000], "w"), (4100, 4096, 8, [1000, 2000, 0, 1000], "f"),
    (64, 4096, 4096, [1, 0, 63], "fd"), (300, 65536, 16, [100, 7, 150], "f"), (520, 8200, 1032, [300, 200], "f"), (520, 1032, 8200, [17, 503], "d"),
    (20000, 272, 1696, [7000, 0, 12000, 900], "w")])
def test_parts_of_a_long_contraction(gl, rows, k, n, sizes, parts):
    lib = load_package()._native.load()
    m, g = rows, len(sizes)
    assert ("f" in parts) == (lib.mi355_w8a8_bf16_grouped_workspace_bytes(m, k, n, g, 0) > 0)
    assert ("d" in parts) == (lib.mi355_w8a8_bf16_grouped_bwd_workspace_bytes(m, k, n, g, 0, 1, 0) > 0)
    assert ("w" in parts) == (lib.mi355_w8a8_bf16_grouped_bwd_workspace_bytes(m, k, n, g, 0, 0, 1) > 0)
    assert lib.mi355_w8a8_bf16_grouped_workspace_bytes(m, k, n, g, 16) == 0
    x, w, dy, st = make(rows, k, n, sizes, seed=5)
    check(gl, x, w, dy, st, sizes)
    check(gl, x, w, dy, st, sizes, torch.float32)
    first = gl.grouped_matmul(x, w, st), *gl.grouped_matmul_backward(x, dy, w, st)
    assert all(torch.equal(a, b) for a, b in zip(first, (gl.grouped_matmul(x, w, st), *gl.grouped_matmul_backward(x, dy, w, st))))
    if sum(sizes) < rows:
        assert not first[0][sum(sizes):].any() and not first[1][sum(sizes):].any()


@pytest.mark.parametrize("flags", [0, 4, 8, 16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_of_other_rows_stay_there(gl, bad, flags):
    """A NaN or infinity in one group's rows or weight, or in rows of no group, reaches that group's results alone, also where K and
    the rows end inside a tile."""
    sizes = [30, 50, 0, 20]
    x, w, dy, st = make(120, 40, 72, sizes)
    want, (wdx, wdw) = gl.grouped_matmul(x, w, st, flags=flags), gl.grouped_matmul_backward(x, dy, w, st, flags=flags)
    x[30:80], dy[30:80], w[1], w[2] = bad, bad, bad, bad
    x[100:], dy[100:] = bad, bad
    out, (dx, dw) = gl.grouped_matmul(x, w, st, flags=flags), gl.grouped_matmul_backward(x, dy, w, st, flags=flags)
    for got, ref in ((out, want), (dx, wdx)):
        assert torch.equal(got[:30], ref[:30]) and torch.equal(got[80:], ref[80:]) and not torch.isfinite(got[30:80]).any()
        assert not got[100:].any()
    assert torch.equal(dw[0], wdw[0]) and torch.equal(dw[2:], wdw[2:]) and not torch.isfinite(dw[1]).any() and not dw[2].any()


def test_differences(gl):
    """Small whole numbers: every sum is exact in bf16, so a change of one value changes the output by the gradient times the change."""
    sizes = [3, 0, 6, 2]
    g = torch.Generator(device=DEV).manual_seed(5)
    ints = lambda *s: torch.randint(-1, 2, s, generator=g, device=DEV).to(torch.bfloat16)
    x, w, dy = ints(13, 16), ints(4, 16, 24), ints(13, 24)
    st = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    dx, dw = gl.grouped_matmul_backward(x, dy, w, st)
    base = gl.grouped_matmul(x, w, st).double()
    for i, c in ((0, 0), (2, 15), (3, 7), (10, 3), (12, 2)):
        moved = x.clone()
        moved[i, c] += 1
        assert float(((gl.grouped_matmul(moved, w, st).double() - base) * dy.double()).sum()) == float(dx[i, c])
    for e, r, c in ((0, 0, 0), (1, 5, 5), (2, 15, 23), (3, 8, 1)):
        moved = w.clone()
        moved[e, r, c] += 1
        assert float(((gl.grouped_matmul(x, moved, st).double() - base) * dy.double()).sum()) == float(dw[e, r, c])


def test_autograd_strides_and_offsets(gl):
    sizes = [20, 0, 45]
    x, w, dy, st = make(70, 48, 56, sizes)
    want = gl.grouped_matmul(x, w, st), *gl.grouped_matmul_backward(x, dy, w, st)
    wide = torch.zeros(70, 96, dtype=torch.bfloat16, device=DEV)
    wide[:, ::2] = x
    xs = wide[:, ::2].requires_grad_()
    buffer = torch.empty(w.numel() + 3, dtype=torch.bfloat16, device=DEV)
    ws = buffer[3:].view_as(w).copy_(w).detach().requires_grad_()
    out = gl.bf16_grouped_linear(xs, ws, st.long())
    out.backward(dy.t().contiguous().t())
    assert torch.equal(out, want[0]) and torch.equal(xs.grad, want[1]) and torch.equal(ws.grad, want[2])
    only_w = w.clone().requires_grad_()
    gl.bf16_grouped_linear(x, only_w, st).backward(dy)
    assert torch.equal(only_w.grad, want[2])
    only_x = x.clone().requires_grad_()
    gl.bf16_grouped_linear(only_x, w, st).backward(dy)
    assert torch.equal(only_x.grad, want[1])


def test_graph_replays_with_other_sizes_and_streams(gl):
    sizes = [33, 60, 7]
    x, w, dy, st = make(100, 64, 96, sizes)
    other = torch.tensor([0, 90, 5], dtype=torch.int32, device=DEV)
    want = {}
    for key, s in (("a", st.clone()), ("b", other)):
        want[key] = gl.grouped_matmul(x, w, s), *gl.grouped_matmul_backward(x, dy, w, s)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = gl.grouped_matmul(x, w, other)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(side, want["b"][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gl.grouped_matmul(x, w, st)
        dx, dw = gl.grouped_matmul_backward(x, dy, w, st)
    for key, s in (("b", other), ("a", torch.tensor(sizes, dtype=torch.int32, device=DEV)), ("b", other)):
        st.copy_(s)
        graph.replay()
        eager = gl.grouped_matmul(x, w, st)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[key][0])
        for got, ref in zip((out, dx, dw), want[key]):
            assert torch.equal(got, ref)


def test_same_bits_at_every_call(gl):
    sizes = [700, 0, 1200, 100]
    x, w, dy, st = make(2048, 256, 384, sizes)
    first = gl.grouped_matmul(x, w, st), *gl.grouped_matmul_backward(x, dy, w, st, dw_dtype=torch.float32)
    for _ in range(3):
        again = gl.grouped_matmul(x, w, st), *gl.grouped_matmul_backward(x, dy, w, st, dw_dtype=torch.float32)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("k,n", [(4096, 8), (8, 4096)])
def test_rows_beyond_32_bits(gl, k, n):
    """The last of 600000 rows lie 4.9 GB behind the first; small whole numbers, whose sums are exact."""
    rows, sizes = 600000, [1, 299999, 0, 299000]
    print(f"[case] {rows} rows, {k} -> {n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(7)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g, device=DEV, dtype=torch.int8).to(torch.bfloat16)
    x, dy, w, st = whole(rows, k), whole(rows, n), whole(4, k, n), torch.tensor(sizes, dtype=torch.int32, device=DEV)
    out = gl.grouped_matmul(x, w, st)
    dx, _ = gl.grouped_matmul_backward(x, dy, w, st, need_dw=False)
    for r, e in ((slice(0, 1), 0), (slice(299990, 300000), 1), (slice(300000, 300010), 3), (slice(598990, 599000), 3)):
        assert torch.equal(out[r].double(), (x[r].double() @ w[e].double()).to(torch.bfloat16).double())
        assert torch.equal(dx[r].double(), (dy[r].double() @ w[e].double().T).to(torch.bfloat16).double())
    assert not out[599000:].any() and not dx[599000:].any()
    _, dw = gl.grouped_matmul_backward(x, dy, w, st, need_dx=False, dw_dtype=torch.float32)  # (at most 1.2 million: exact)
    assert torch.equal(dw[3], x[300000:599000].float().T @ dy[300000:599000].float()) and not dw[2].any()


def test_weights_beyond_32_bits(gl):
    """The last of 70 groups lie 4.6 GB behind the first."""
    groups, k, n, rows = 70, 4096, 8192, 140
    print(f"[case] {groups} groups, {k} -> {n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(8)
    x, dy = (torch.randn(rows, c, generator=g, device=DEV).to(torch.bfloat16) for c in (k, n))
    w = torch.empty(groups, k, n, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    sizes = torch.full((groups,), 2, dtype=torch.int32, device=DEV)
    sizes[40], sizes[69] = 0, 4
    out = gl.grouped_matmul(x, w, sizes)
    dx, dw = gl.grouped_matmul_backward(x, dy, w, sizes)
    for e, r in ((0, slice(0, 2)), (66, slice(130, 132)), (69, slice(136, 140))):
        xd, dd, wd = x[r].double(), dy[r].double(), w[e].double()
        close(out[r], xd @ wd, xd.abs() @ wd.abs(), k)
        close(dx[r], dd @ wd.T, dd.abs() @ wd.abs().T, n)
        close(dw[e], xd.T @ dd, xd.abs().T @ dd.abs(), 4)
    assert not dw[40].any()


def test_the_most_groups_and_rows(gl):
    sizes = torch.full((1024,), 1023, dtype=torch.int32, device=DEV)
    sizes[1000] = 0
    rows = 1 << 20
    x, dy = (torch.randint(-1, 2, (rows, 8), device=DEV, dtype=torch.int8).to(torch.bfloat16) for _ in range(2))
    w = torch.randint(-1, 2, (1024, 8, 8), device=DEV, dtype=torch.int8).to(torch.bfloat16)
    group = torch.repeat_interleave(torch.arange(1024, device=DEV), sizes.long())
    held = group.numel()
    want = (x[:held, :, None].float() * w[group].float()).sum(1)
    out = gl.grouped_matmul(x, w, sizes)
    assert torch.equal(out[:held].float(), want) and not out[held:].any()
    dx, dw = gl.grouped_matmul_backward(x, dy, w, sizes, dw_dtype=torch.float32)
    assert torch.equal(dx[:held].float(), (dy[:held, None, :].float() * w[group].float()).sum(2)) and not dx[held:].any()
    outer = torch.zeros(1024, 8, 8, device=DEV).index_add_(0, group, x[:held, :, None].float() * dy[:held, None, :].float())  # (whole numbers: exact)
    assert torch.equal(dw, outer)
    with pytest.raises(ValueError, match="at most"):
        gl.grouped_matmul(torch.zeros(rows + 1, 8, dtype=torch.bfloat16, device=DEV), w, sizes)


@pytest.mark.parametrize("native", [True, False])
def test_wanted_gradients_go_by_truth(gl, monkeypatch, native):
    """Whole numbers and NumPy's truth values say what True and False say, through the host module and without it."""
    if not native:
        monkeypatch.setattr(load_package()._native, "host", lambda: None)
    x, w, dy, st = make(50, 64, 40, [20, 0, 25])
    dx, dw = gl.grouped_matmul_backward(x, dy, w, st)
    for want_dx, want_dw in ((1, 1), (1, 0), (0, 1), (True, 1), (2, False), (numpy.True_, numpy.True_), (numpy.True_, numpy.False_), (numpy.bool_(0), numpy.bool_(1))):
        got = gl.grouped_matmul_backward(x, dy, w, st, need_dx=want_dx, need_dw=want_dw)
        for value, ref, wanted in zip(got, (dx, dw), (want_dx, want_dw)):
            assert torch.equal(value, ref) if wanted else value is None, (want_dx, want_dw)
    assert gl.grouped_matmul_backward(x, dy, w, st, need_dx=0, need_dw=numpy.False_) == (None, None)
