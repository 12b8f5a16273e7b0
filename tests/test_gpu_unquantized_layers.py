"""Layers that keep bf16 weights, alone and together: a LoRA embedding, experts, and the clipping of their adapters' gradients.

Tolerances count the roundings to bf16 on the way, half a step (2^-8 of the value) each: a value behind c of them is off by at most
about c * 2^-8 of the sum of its terms' magnitudes; float32 sums add less than 2^-12 of it at these sizes (at most 2000 terms)."""

import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
STEP = 2.0 ** -8


@pytest.fixture(scope="module")
def lora():
    return load_package().lora


def fill(layer, g):
    layer.lora_A = (torch.randn(layer.lora_A.shape, generator=g, device=DEV) * 0.3).to(BF16).requires_grad_()
    layer.lora_B = (torch.randn(layer.lora_B.shape, generator=g, device=DEV) * 0.3).to(BF16).requires_grad_()
    layer.lora_scaling = torch.rand(layer.max_lora_adapters, generator=g, device=DEV) + 0.5


def off_by(got, want, magnitudes, roundings):
    return float(((got.detach().double() - want).abs() - roundings * STEP * magnitudes - 2.0 ** -12 * magnitudes).max())


@pytest.mark.parametrize("n_ad,rank,vocab,width,batch,length", [
    (0, 8, 50, 24, 2, 3), (1, 8, 997, 64, 3, 7), (3, 4, 997, 136, 5, 11), (4, 20, 30000, 256, 16, 1), (8, 32, 1000, 512, 9, 50)])
def test_embed(lora, n_ad, rank, vocab, width, batch, length):
    print(f"[case] {n_ad} adapters of rank {rank}, {vocab} x {width}, {batch} x {length}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    layer = lora.LoRAEmbed(vocab, width, embedding=torch.randn(vocab, width, generator=g, device=DEV), max_lora_adapters=n_ad, max_lora_rank=rank)
    ids = torch.randint(0, vocab, (batch, length), generator=g, device=DEV)
    ids[0] = ids[-1, 0]
    table = layer.embedding.double()[ids]
    assert torch.equal(layer(ids), layer.embedding[ids])
    if not n_ad:
        return
    fill(layer, g)
    index = torch.randint(0, n_ad, (batch,), generator=g, device=DEV)
    layer.embedding.requires_grad_()
    out = layer(ids, index)
    a, b, s = layer.lora_A.detach().double(), layer.lora_B.detach().double(), layer.lora_scaling.double()
    z = a[index[:, None], ids] * s[index][:, None, None]
    want = table + torch.matmul(z, b[index])
    mags = table.abs() + torch.matmul(z.abs(), b[index].abs())
    assert off_by(out, want, mags, 3) <= 0  # z, the product, the sum
    dy = torch.randn(out.shape, generator=g, device=DEV).to(BF16)
    out.backward(dy)
    d = dy.double()
    want_a, mags_a = torch.zeros_like(a), torch.zeros_like(a)
    want_b, mags_b = torch.zeros_like(b), torch.zeros_like(b)
    for i in range(batch):
        k = int(index[i])
        want_a[k].index_add_(0, ids[i], s[k] * (d[i] @ b[k].T))
        mags_a[k].index_add_(0, ids[i], s[k] * (d[i].abs() @ b[k].abs().T))
        want_b[k] += z[i].T @ d[i]
        mags_b[k] += z[i].abs().T @ d[i].abs()
    assert off_by(layer.lora_A.grad, want_a, mags_a, 2) <= 0  # dz, the row's sum
    assert off_by(layer.lora_B.grad, want_b, mags_b, 2) <= 0  # z, the sum
    want_t = torch.zeros_like(layer.embedding, dtype=torch.float64).index_add_(0, ids.reshape(-1), d.reshape(-1, width))
    mags_t = torch.zeros_like(want_t).index_add_(0, ids.reshape(-1), d.abs().reshape(-1, width))
    assert off_by(layer.embedding.grad, want_t, mags_t, 1) <= 0


@pytest.mark.parametrize("n_exp,n_ad,k,n,rank,sizes", [(4, 2, 64, 96, 8, [5, 0, 9, 3]), (5, 3, 72, 40, 12, [20, 1, 0, 30, 7]), (2, 1, 128, 64, 4, [3, 0])])
def test_dense_experts(lora, n_exp, n_ad, k, n, rank, sizes):
    print(f"[case] {n_exp} experts, {n_ad} adapters, {k} -> {n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(4)
    layer = lora.LoRAExpert(n_exp, k, n, max_lora_adapters=n_ad, max_lora_rank=rank)
    layer.load_unquantized(torch.randn(n_exp, k, n, generator=g, device=DEV) * k ** -0.5)
    fill(layer, g)
    rows = sum(sizes) + 2  # (two rows of no expert)
    x = torch.randn(rows, k, generator=g, device=DEV).to(BF16).requires_grad_()
    st = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    index = torch.randint(0, n_ad, (rows,), generator=g, device=DEV)
    layer.unquantized.requires_grad_()
    plain, out = layer(x, st), layer(x, st, index)
    expert = torch.repeat_interleave(torch.arange(n_exp, device=DEV), st.long())
    held = expert.numel()
    xd, w = x.detach().double()[:held], layer.unquantized.detach().double()[expert]
    a, b = layer.lora_A.detach().double()[index[:held], expert], layer.lora_B.detach().double()[index[:held], expert]
    s = layer.lora_scaling.double()[index[:held]][:, None]
    mul = lambda v, m: torch.matmul(v[:, None], m)[:, 0]
    base, base_m = mul(xd, w), mul(xd.abs(), w.abs())
    z, z_m = s * mul(xd, a), s * mul(xd.abs(), a.abs())
    assert off_by(plain[:held], base, base_m, 1) <= 0 and not plain[held:].any() and not out[held:].any()
    mags = base_m + mul(z_m, b.abs())
    assert off_by(out[:held], base + mul(z, b), mags, 4) <= 0  # z, scaled z, the product, the sum
    dy = torch.randn(out.shape, generator=g, device=DEV).to(BF16)
    out.backward(dy)
    d = dy.double()[:held]
    t = lambda m: m.transpose(1, 2)
    dz, dz_m = s * mul(d, t(b)), s * mul(d.abs(), t(b).abs())
    assert off_by(x.grad[:held], mul(d, t(w)) + mul(dz, t(a)), mul(d.abs(), t(w).abs()) + mul(dz_m, t(a).abs()), 4) <= 0
    assert not x.grad[held:].any()
    outer = lambda u, v: u[:, :, None] * v[:, None, :]
    spot = index[:held] * n_exp + expert
    sum_of = lambda terms, count, at: torch.zeros(count, *terms.shape[1:], dtype=torch.float64, device=DEV).index_add_(0, at, terms)
    pairs = n_ad * n_exp
    assert off_by(layer.lora_A.grad.reshape(pairs, k, rank), sum_of(outer(xd, dz), pairs, spot), sum_of(outer(xd.abs(), dz_m), pairs, spot), 3) <= 0
    assert off_by(layer.lora_B.grad.reshape(pairs, rank, n), sum_of(outer(z, d), pairs, spot), sum_of(outer(z_m, d.abs()), pairs, spot), 3) <= 0
    assert off_by(layer.unquantized.grad, sum_of(outer(xd, d), n_exp, expert), sum_of(outer(xd.abs(), d.abs()), n_exp, expert), 1) <= 0


def test_a_training_step(lora):
    """Embedding, routing, experts, loss, gradients, clipping: the clipped gradients are those of the backward times each adapter's factor,
    and a second step from the same state gives the same bits."""
    pkg = load_package()
    g = torch.Generator(device=DEV).manual_seed(5)
    n_ad, n_exp, top_k, hidden = 3, 8, 2, 64
    embed = lora.LoRAEmbed(500, hidden, embedding=torch.randn(500, hidden, generator=g, device=DEV), max_lora_adapters=n_ad, max_lora_rank=8)
    up = lora.LoRAExpert(n_exp, hidden, 96, max_lora_adapters=n_ad, max_lora_rank=8)
    up.load_unquantized(torch.randn(n_exp, hidden, 96, generator=g, device=DEV) * 0.1)
    for layer in (embed, up):
        fill(layer, g)
    ids = torch.randint(0, 500, (6, 13), generator=g, device=DEV)
    index = torch.tensor([0, 1, 2, 0, 0, 1], dtype=torch.int32, device=DEV)
    router = torch.randn(hidden, n_exp, generator=g, device=DEV)

    def step():
        for layer in (embed, up):
            layer.lora_A.grad = layer.lora_B.grad = None
        h = embed(ids, index).reshape(-1, hidden)
        _, selected = pkg.w8a8_lora.moe_route(h.detach().float() @ router, top_k)
        _, sizes, order, _, sorted_adapters = pkg.w8a8_lora.moe_dispatch(None, selected, n_exp, repeat=top_k, adapter_indices=index.repeat_interleave(13))
        y = up(h[(order // top_k).long()], sizes, sorted_adapters)
        y.float().square().mean().backward()
        return [p.grad.clone() for layer in (embed, up) for p in (layer.lora_A, layer.lora_B)]

    before = step()
    norms = torch.stack([b.double().flatten(1).square().sum(1) for b in before]).sum(0).sqrt()
    limits = (norms * torch.tensor([0.5, 2.0, 0.9], device=DEV)).float()
    got = lora.clip_adapter_gradients([embed, up], limits)
    assert bool(((got.double() - norms).abs() <= norms * 2.0 ** -23).all())
    after = [p.grad.clone() for layer in (embed, up) for p in (layer.lora_A, layer.lora_B)]
    for b, a in zip(before, after):
        assert torch.equal(a[1], b[1])  # below its limit
        for k, f in ((0, 0.5), (2, 0.9)):
            want = b[k].double() * f
            assert bool(((a[k].double() - want).abs() <= (STEP + 2.0 ** -22) * want.abs() + 1e-40).all())
    assert all(torch.equal(a, b) for a, b in zip(before, step()))
    assert all(b.abs().sum() > 0 for b in before)


def test_refusals(lora):
    layer = lora.LoRAEmbed(10, 16, max_lora_adapters=2)
    with pytest.raises(RuntimeError, match="load_unquantized"):
        layer(torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="table"):
        layer.load_unquantized(torch.zeros(10, 8, device=DEV))
    layer.load_unquantized(torch.zeros(10, 16, device=DEV))
    with pytest.raises(ValueError, match="one entry per example"):
        layer(torch.zeros(2, 3, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="no|none"):
        lora.clip_adapter_gradients([layer], 1.0)
    with pytest.raises(ValueError, match="kernels"):
        lora.LoRAExpert(2, 8, 8).load_unquantized(torch.zeros(2, 8, 16, device=DEV))
    with pytest.raises(TypeError, match="integers"):
        layer(torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, device=DEV))
    for bad in (torch.zeros((), dtype=torch.int32, device=DEV), torch.zeros((2, 1), dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError, match="one entry per example"):
            layer(torch.zeros(2, dtype=torch.int64, device=DEV), bad)


def test_adapters_and_ids_out_of_range(lora):
    g = torch.Generator(device=DEV).manual_seed(6)
    for n_ad in (1, 3):
        layer = lora.LoRAEmbed(40, 16, embedding=torch.randn(40, 16, generator=g, device=DEV), max_lora_adapters=n_ad)
        fill(layer, g)
        ids = torch.tensor([[3, 4], [5, 6], [7, 40], [-1, 8]], device=DEV)
        out = layer(ids, torch.tensor([-1, 2 ** 32, n_ad, n_ad - 1], device=DEV))
        want = layer.embedding[ids.clamp(0, 39)] * ((ids >= 0) & (ids < 40))[..., None]
        assert torch.equal(out[:3], want[:3]) and torch.equal(out[3, 0], want[3, 0]) and not torch.equal(out[3, 1], want[3, 1])
        out.float().sum().backward()
        used = torch.zeros(n_ad, 40, dtype=torch.bool, device=DEV)
        used[n_ad - 1, 8] = True
        assert torch.equal(layer.lora_A.grad.any(-1), used)
        assert torch.equal(layer.lora_B.grad.flatten(1).any(1), used.any(1))


def test_new_adapters_leave_the_layers_as_they_are(lora):
    g = torch.Generator(device=DEV).manual_seed(7)
    embed = lora.LoRAEmbed(90, 24, embedding=torch.randn(90, 24, generator=g, device=DEV), max_lora_adapters=2, max_lora_rank=8)
    experts = lora.LoRAExpert(4, 24, 32, max_lora_adapters=2, max_lora_rank=8)
    experts.load_unquantized(torch.randn(4, 24, 32, generator=g, device=DEV))
    for layer, rank in ((embed, 6), (experts, 16)):
        lora.init_lora_adapter(layer, 1, rank=rank, alpha=16.0)
        kept = rank if layer is embed else rank // 4
        assert layer.lora_A[1, ..., :kept].any() and not layer.lora_A[1, ..., kept:].any() and not layer.lora_A[0].any()
        assert abs(float(layer.lora_scaling[1]) - 16.0 / kept) <= 2.0 ** -24 * 16.0 / kept  # (16 / 6 rounds to float32 by at most half a step)
    ids, index = torch.arange(12, device=DEV), torch.arange(12, device=DEV) % 2
    assert torch.equal(embed(ids, index), embed(ids))
    sizes = torch.tensor([3, 3, 3, 3], dtype=torch.int32, device=DEV)
    x = torch.randn(12, 24, generator=g, device=DEV).to(BF16)
    assert torch.equal(experts(x, sizes, index), experts(x, sizes))


def test_a_captured_backward(lora):
    """Forward, gradients and clipping of an embedding and its product in one graph, replayed with other ids and sizes while the program works
    on; two graphs with buffers of their own take turns."""
    pkg = load_package()
    gl, em, gc = pkg.bf16_grouped_linear, pkg.embedding, pkg.grad_clip
    g = torch.Generator(device=DEV).manual_seed(8)
    n_ad, vocab, rank, width, rows = 3, 300, 8, 64, 200
    a = (torch.randn(n_ad, vocab, rank, generator=g, device=DEV)).to(BF16).requires_grad_()
    b = (torch.randn(n_ad, rank, width, generator=g, device=DEV)).to(BF16).requires_grad_()

    class Step:
        def __init__(self):
            self.ids = torch.zeros(rows, dtype=torch.int64, device=DEV)
            self.index = torch.zeros(rows, dtype=torch.int32, device=DEV)
            self.sizes = torch.zeros(n_ad, dtype=torch.int32, device=DEV)
            self.dy = torch.zeros(rows, width, dtype=BF16, device=DEV)

        def fill(self):
            self.ids.copy_(torch.randint(0, vocab, (rows,), generator=g, device=DEV))
            self.index.copy_(torch.randint(0, n_ad, (rows,), generator=g, device=DEV).sort().values)
            self.sizes.copy_(torch.bincount(self.index, minlength=n_ad))
            self.dy.copy_(torch.randn(rows, width, generator=g, device=DEV))

        def run(self):
            y = gl.bf16_grouped_linear(em.embed(a, self.ids, 0.5, adapter_indices=self.index), b, self.sizes)
            da, db = torch.autograd.grad(y, (a, b), self.dy)
            (da, db), norms = gc.clip_grad_norm([da, db], 1.0, per_adapter=True)
            return y.detach(), da, db, norms

        def run_into_leaves(self):
            a.grad = b.grad = None
            gl.bf16_grouped_linear(em.embed(a, self.ids, 0.5, adapter_indices=self.index), b, self.sizes).backward(self.dy)
            return a.grad, b.grad

    first, second, third = Step(), Step(), Step()
    graphs = []
    for step, call in ((first, Step.run), (second, Step.run), (third, Step.run_into_leaves)):
        step.fill()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(step)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = call(step)
        graphs.append((step, call, graph, results))
    for turn in range(4):
        for step, call, graph, results in graphs:
            step.fill()
            graph.replay()
            got = [t.clone() for t in results]
            kept = a.grad, b.grad
            want = call(step)
            a.grad, b.grad = kept
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (turn, call.__name__)


def test_host_module_and_general_path_agree(monkeypatch):
    pkg = load_package()
    gl, em = pkg.bf16_grouped_linear, pkg.embedding
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(100, 72, generator=g, device=DEV).to(BF16)
    w = torch.randn(5, 72, 136, generator=g, device=DEV).to(BF16)
    dy = torch.randn(100, 136, generator=g, device=DEV).to(BF16)
    sizes = torch.tensor([10, 0, 50, 7, 20], dtype=torch.int32, device=DEV)
    table = torch.randn(3, 50, 40, generator=g, device=DEV)
    ids = torch.randint(0, 50, (10, 6), generator=g, device=DEV)
    index = torch.randint(0, 3, (10,), generator=g, device=DEV)
    scales = torch.rand(3, generator=g, device=DEV)
    d = torch.randn(10, 6, 40, generator=g, device=DEV)

    def calls():
        out = [gl.grouped_matmul(x, w, sizes), gl.grouped_matmul(x[::2], w, sizes.long()), gl.grouped_matmul(x, w.transpose(0, 1).contiguous().transpose(0, 1), sizes)]
        for dtype in (BF16, torch.float32):
            out += gl.grouped_matmul_backward(x, dy, w, sizes, dw_dtype=dtype)
        out += [gl.grouped_matmul_backward(None, dy, w, sizes, need_dw=False)[0], gl.grouped_matmul_backward(x, dy, None, sizes, need_dx=False)[1]]
        for t, e in ((table, d), (table.to(BF16), d.to(BF16))):
            for i, n in ((ids, index), (ids.int(), index.int()), (ids, index.repeat_interleave(6))):
                out += [em.lookup(t, i, scales, adapter_indices=n), em.lookup_backward(e, i, t.shape, scales, adapter_indices=n)]
            out += [em.lookup(t[0], ids), em.lookup_backward(e, ids, t[0].shape, 2.0), em.lookup(t[0, :, 1:], ids, 0.5)]
            out += [em.lookup_backward(e.transpose(0, 1).contiguous().transpose(0, 1), ids, t[0].shape, -1.0)]
        return out

    first = calls()
    monkeypatch.setattr(pkg._native, "host", lambda: None)
    for i, (one, other) in enumerate(zip(first, calls())):
        assert one.dtype == other.dtype and torch.equal(one, other), i


def test_other_streams(lora):
    """Operands made on one stream, used on another behind a wait, with the side stream's own results."""
    g = torch.Generator(device=DEV).manual_seed(10)
    layer = lora.LoRAEmbed(700, 64, embedding=torch.randn(700, 64, generator=g, device=DEV), max_lora_adapters=4)
    fill(layer, g)
    ids = torch.randint(0, 700, (8, 300), generator=g, device=DEV)
    index = torch.randint(0, 4, (8,), generator=g, device=DEV)
    dy = torch.randn(8, 300, 64, generator=g, device=DEV).to(BF16)

    def step():
        out = layer(ids, index)
        return (out.detach(), *torch.autograd.grad(out, (layer.lora_A, layer.lora_B), dy))

    want = step()
    sides = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for other in got for a, b in zip(want, other))


def test_second_derivatives_are_refused():
    pkg = load_package()
    x = torch.randn(4, 8, device=DEV).to(BF16).requires_grad_()
    w = torch.randn(1, 8, 8, device=DEV).to(BF16).requires_grad_()
    dx, = torch.autograd.grad(pkg.bf16_grouped_linear.bf16_grouped_linear(x, w, torch.tensor([4], device=DEV)).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().sum().backward()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32])
def test_whole_numbers_of_any_width(lora, dtype):
    """Adapters and sizes of narrow types give what int64 ones give, forward and backward."""
    pkg = load_package()
    g = torch.Generator(device=DEV).manual_seed(11)
    layer = lora.LoRAEmbed(50, 24, embedding=torch.randn(50, 24, generator=g, device=DEV), max_lora_adapters=3)
    fill(layer, g)
    ids, index = torch.randint(0, 50, (6, 5), generator=g, device=DEV), torch.tensor([0, 2, 1, 1, 0, 2], device=DEV)
    dy = torch.randn(6, 5, 24, generator=g, device=DEV).to(BF16)

    def of(index):
        out = layer(ids, index)
        return out.detach(), *torch.autograd.grad(out, (layer.lora_A, layer.lora_B), dy)

    want = of(index)
    assert all(torch.equal(a, b) for a, b in zip(want, of(index.to(dtype)))) and not torch.equal(want[0], layer(ids).detach()) and want[1].any()
    if dtype.is_signed:
        assert torch.equal(layer(ids, torch.full((6,), -1, dtype=dtype, device=DEV)), layer(ids))
    em, gl = pkg.embedding, pkg.bf16_grouped_linear
    assert torch.equal(em.lookup(layer.lora_A, ids, 2.0, adapter_indices=index.to(dtype)), em.lookup(layer.lora_A, ids, 2.0, adapter_indices=index))
    sizes = torch.tensor([100, 0, 127], device=DEV)
    x, w = torch.randn(40000, 16, generator=g, device=DEV).to(BF16), torch.randn(3, 16, 24, generator=g, device=DEV).to(BF16)
    assert torch.equal(gl.grouped_matmul(x, w, sizes.to(dtype)), gl.grouped_matmul(x, w, sizes))
    experts = lora.LoRAExpert(3, 16, 24, max_lora_adapters=3)
    experts.load_unquantized(w)
    fill(experts, g)
    adapters = torch.randint(0, 3, (40000,), generator=g, device=DEV)
    assert torch.equal(experts(x, sizes.to(dtype), adapters.to(dtype)), experts(x, sizes, adapters))


@pytest.mark.parametrize("n_ad", [1, 3, 1024])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_infinities_beside_adapters_and_ids_out_of_range(lora, n_ad, bad):
    """A token without an adapter or a row has no part in the adapters' term: infinities of B do not reach its row, those of its gradient neither A nor B."""
    g = torch.Generator(device=DEV).manual_seed(12)
    layer = lora.LoRAEmbed(40, 16, embedding=torch.randn(40, 16, generator=g, device=DEV), max_lora_adapters=n_ad)
    fill(layer, g)
    ids = torch.tensor([[3, 4], [5, 6], [7, 40], [-1, 8]], device=DEV)
    index = torch.tensor([-1, 2 ** 32, n_ad, n_ad - 1], device=DEV)
    dy = torch.randn(4, 2, 16, generator=g, device=DEV).to(BF16)
    held = torch.zeros(4, 2, dtype=torch.bool, device=DEV)
    held[3, 1] = True
    out = layer(ids, index)
    want = torch.autograd.grad(out, (layer.lora_A, layer.lora_B), dy)
    got = torch.autograd.grad(layer(ids, index), (layer.lora_A, layer.lora_B), torch.where(held[..., None], dy, bad))
    assert all(torch.equal(a, b) and torch.isfinite(a).all() and a.any() for a, b in zip(got, want))
    layer.lora_B.data[...] = bad
    other = layer(ids, index)
    assert torch.equal(other[~held], out[~held]) and torch.equal(other[~held], layer(ids)[~held]) and not torch.isfinite(other[held]).any()


def test_streams_of_living_graphs(monkeypatch):
    """The rule for captured backward passes with streams as they are and captures that are only claimed: no graph that lives, ours or another
    operation's, may have brought the default stream to a leaf; any other stream may be there."""
    gl = load_package().bf16_grouped_linear
    x, w = torch.ones(8, 8, dtype=BF16, device=DEV), torch.ones(1, 8, 8, dtype=BF16, device=DEV).requires_grad_()
    sizes = torch.tensor([8], dtype=torch.int32, device=DEV)
    ours, theirs, side = lambda: gl.bf16_grouped_linear(x, w, sizes), lambda: (w * 2).sum(), torch.cuda.Stream()

    def on_side(call):
        with torch.cuda.stream(side):
            return call()

    def captured():
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            with torch.cuda.stream(torch.cuda.Stream()):
                return torch.autograd.grad(gl.bf16_grouped_linear(x, w, sizes).sum(), w)

    captured()
    for call in (ours, theirs):
        graph = call()
        with pytest.raises(RuntimeError, match="lives"):
            captured()
        later = on_side(ours)
        del graph
        with pytest.raises(RuntimeError, match="lives"):  # (a graph of the side stream keeps what the default one's made)
            captured()
        del later
        captured()
        graph = on_side(call)
        captured()
        later = call()
        captured()
        del graph
        captured()
        del later
    torch.cuda.synchronize()


@pytest.mark.parametrize("kept", [False, True])
def test_a_capture_beside_the_last_warm_up(lora, kept):
    """A training step warmed up on a side stream and captured while its last output still lives, its gradients new or (kept) added to the ones that
    are there; replays with other inputs give what an eager step of the same weights gives."""
    g = torch.Generator(device=DEV).manual_seed(13)
    embed = lora.LoRAEmbed(300, 64, embedding=torch.randn(300, 64, generator=g, device=DEV), max_lora_adapters=3, max_lora_rank=8)
    fill(embed, g)
    head = torch.randn(1, 64, 96, generator=g, device=DEV).to(BF16).requires_grad_()
    ids = torch.randint(0, 300, (6, 20), generator=g, device=DEV)
    index = torch.randint(0, 3, (6,), generator=g, device=DEV)
    target = torch.randn(120, 96, generator=g, device=DEV).to(BF16)
    sizes = torch.tensor([120], dtype=torch.int32, device=DEV)
    gl = load_package().bf16_grouped_linear
    leaves = [embed.lora_A, embed.lora_B, head]
    twins = [t.detach().clone().requires_grad_() for t in leaves]

    def step(a, b, w):
        embed.lora_A, embed.lora_B = a, b
        for p in (a, b, w):
            if kept and p.grad is not None:
                p.grad.zero_()
            else:
                p.grad = None
        out = gl.bf16_grouped_linear(embed(ids, index).reshape(-1, 64), w, sizes)
        out.backward(target)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            last = step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*leaves)
    grads = [p.grad for p in leaves]
    assert last.grad_fn is not None
    for turn in range(4):
        ids.copy_(torch.randint(0, 300, ids.shape, generator=g, device=DEV))
        index.copy_(torch.randint(0, 3, index.shape, generator=g, device=DEV))
        target.copy_(torch.randn(target.shape, generator=g, device=DEV))
        graph.replay()
        got = [t.detach().clone() for t in (captured, *grads)]
        want = step(*twins)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (want.detach(), *(p.grad for p in twins)))), turn


def test_streams_of_living_graphs_behind_other_operations(lora, monkeypatch):
    """The same rule for leaves that reach the products through other operations: a view, a sum, adapters whose rank is filled up, a graph in between."""
    gl = load_package().bf16_grouped_linear
    x, sizes = torch.ones(8, 8, dtype=BF16, device=DEV), torch.tensor([8], dtype=torch.int32, device=DEV)
    w, v = (torch.ones(1, 8, 8, dtype=BF16, device=DEV).requires_grad_() for _ in range(2))
    embed = lora.LoRAEmbed(20, 16, embedding=torch.ones(20, 16, device=DEV), max_lora_adapters=2, max_lora_rank=5)
    embed.lora_B.requires_grad_()  # (B alone is trained)
    ids, index = torch.arange(6, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    calls = [(w, lambda: gl.bf16_grouped_linear(x, w.transpose(1, 2), sizes)), (w, lambda: gl.bf16_grouped_linear(x, w + v, sizes)),
             (v, lambda: gl.bf16_grouped_linear(x, w + v, sizes)), (w, lambda: gl.bf16_grouped_linear(gl.bf16_grouped_linear(x, w * 2, sizes), v, sizes)),
             (embed.lora_B, lambda: embed(ids, index))]
    for leaf, call in calls:

        def captured():
            with monkeypatch.context() as m:
                m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
                with torch.cuda.stream(torch.cuda.Stream()):
                    return torch.autograd.grad(call().sum(), leaf)

        captured()
        living = (leaf * 2).sum()
        with pytest.raises(RuntimeError, match="lives"):
            captured()
        del living
        captured()
        torch.cuda.synchronize()
