"""Embedding rows and the table's gradient.

The forward is one float32 product and one rounding, as elementary torch operations make it: equal bits.  A gradient row is a
float32 sum of c rows (off by at most c * 2^-24 of the magnitudes' sum), times the scale (2^-24), rounded to the type (bf16: half a
step, 2^-8)."""

import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def em():
    return load_package().embedding


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def exact_grad(dy, ids, shape, scale, adapters):
    flat = ids.reshape(-1).long()
    vocab, width = shape[-2:]
    n_ad = shape[0] if len(shape) == 3 else 1
    held = (flat >= 0) & (flat < vocab)
    factor = torch.as_tensor(1.0 if scale is None else scale, dtype=torch.float64, device=DEV).expand(n_ad)
    if adapters is not None:
        a = adapters.long().repeat_interleave(flat.numel() // adapters.numel())
        held &= (a >= 0) & (a < n_ad)
    else:
        a = torch.zeros_like(flat)
    a, flat = a.clamp(0, n_ad - 1), flat.clamp(0, vocab - 1)
    key = (a * vocab + flat)[held]
    d = dy.reshape(-1, width)[held].double()
    grad = torch.zeros(n_ad * vocab, width, dtype=torch.float64, device=DEV).index_add_(0, key, d * factor[a[held], None])
    mags = torch.zeros(n_ad * vocab, width, dtype=torch.float64, device=DEV).index_add_(0, key, d.abs() * factor[a[held], None].abs())
    count = torch.bincount(key, minlength=n_ad * vocab)
    return grad.view(shape), mags.view(shape), count.view(*shape[:-1], 1)


def check_grad(em, dy, ids, shape, scale=None, adapters=None):
    print(f"[case] {tuple(ids.shape)} ids, table {shape}, {dy.dtype}", flush=True)
    got = em.lookup_backward(dy, ids, shape, scale, adapter_indices=adapters)
    want, mags, count = exact_grad(dy, ids, shape, scale, adapters)
    tol = (count + 1) * 2.0 ** -24 * mags + (2.0 ** -8 if dy.dtype == BF16 else 2.0 ** -24) * want.abs()
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(got).any() and float(off.max()) <= 0.0, float(off.max())
    assert not got[(count == 0).expand_as(got)].any()
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab,width,shape,ids_dtype", [
    (1, 1, (1,), torch.int32), (7, 3, (5,), torch.int64), (1000, 8, (3, 17), torch.int32), (513, 65, (40,), torch.int64),
    (50257, 96, (2, 300), torch.int64), (151936, 2560, (16,), torch.int32), (300, 4096, (1,), torch.int32)])
def test_forward(em, dtype, vocab, width, shape, ids_dtype):
    g = gen()
    table = torch.randn(vocab, width, generator=g, device=DEV).to(dtype)
    ids = torch.randint(0, vocab, shape, generator=g, device=DEV, dtype=ids_dtype)
    for scale in (None, 0.7, -3.0):
        want = (table[ids.long()].float() * (1.0 if scale is None else scale)).to(dtype)
        assert torch.equal(em.lookup(table, ids, scale), want)


@pytest.mark.parametrize("n_ad,width", [(1, 32), (3, 5), (8, 32), (16, 64)])
def test_forward_of_adapters(em, n_ad, width):
    g = gen(1)
    table = torch.randn(n_ad, 999, width, generator=g, device=DEV).to(BF16)
    ids = torch.randint(0, 999, (6, 11), generator=g, device=DEV)
    index = torch.randint(0, n_ad, (6,), generator=g, device=DEV)
    scale = torch.rand(n_ad, generator=g, device=DEV) + 0.5
    want = (table[index[:, None], ids].float() * scale[index][:, None, None]).to(BF16)
    assert torch.equal(em.lookup(table, ids, scale, adapter_indices=index), want)
    assert torch.equal(em.lookup(table, ids.int(), scale, adapter_indices=index.int().repeat_interleave(11)), want)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_ids_out_of_range(em, ids_dtype):
    table = torch.randn(2, 10, 24, generator=gen(), device=DEV).to(BF16)
    ids = torch.tensor([0, 9, 10, -1, 5, 2 ** 31 - 1, -2 ** 31, 3], dtype=ids_dtype, device=DEV)
    if ids_dtype == torch.int64:
        ids = torch.cat([ids, torch.tensor([2 ** 32, 2 ** 32 + 3, -2 ** 63], device=DEV)])
    index = torch.zeros(ids.numel(), dtype=torch.int32, device=DEV)
    index[4], index[7] = 2, -1
    out = em.lookup(table, ids, 2.0, adapter_indices=index)
    assert torch.equal(out[:2], (table[0][[0, 9]].float() * 2).to(BF16)) and not out[2:].any()
    check_grad(em, torch.ones(ids.numel(), 24, dtype=BF16, device=DEV), ids, (2, 10, 24), 2.0, index)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab,width,n,hot", [
    (1, 1, 1, 0.0), (1, 8, 1000, 0.0), (11, 3, 29, 0.0), (1000, 8, 8, 0.0), (1000, 8, 9, 0.5), (2047, 33, 1024, 0.3), (2048, 64, 1025, 0.3),
    (50257, 136, 5000, 0.2), (151936, 256, 4097, 0.9), (300, 1000, 2000, 1.0), (97, 24, 70001, 0.1)])
def test_gradient(em, dtype, vocab, width, n, hot):
    g = gen(2)
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    ids[torch.rand(n, generator=g, device=DEV) < hot] = vocab // 2
    dy = torch.randn(n, width, generator=g, device=DEV).to(dtype)
    got = check_grad(em, dy, ids, (vocab, width), 1.7)
    assert torch.equal(got, em.lookup_backward(dy, ids.int(), (vocab, width), 1.7))  # the same bits


@pytest.mark.parametrize("n_ad,vocab,width,n", [(1, 500, 16, 300), (4, 151936, 32, 3000), (16, 1000, 7, 2500), (64, 151936, 8, 9000)])
def test_gradient_of_adapters(em, n_ad, vocab, width, n):
    g = gen(3)
    ids = torch.randint(0, min(vocab, 700), (n,), generator=g, device=DEV)
    index = torch.randint(0, n_ad, (n,), generator=g, device=DEV)
    scale = torch.rand(n_ad, generator=g, device=DEV) + 0.5
    check_grad(em, torch.randn(n, width, generator=g, device=DEV).to(BF16), ids, (n_ad, vocab, width), scale, index)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [5, 9, 15, 513, 3415])
def test_rows_that_begin_anywhere(em, dtype, width):
    """Widths that are no multiple of 16 bytes, from views that begin in the middle of a buffer; the values around them stay."""
    g = gen(7)
    for vocab, n, hot in ((700, 1500, 0.5), (40, 700, 0.0)):
        ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
        ids[torch.rand(n, generator=g, device=DEV) < hot] = 3
        buffer = torch.randn(n * width + 9, generator=g, device=DEV).to(dtype)
        dy = buffer[3:3 + n * width].view(n, width)
        check_grad(em, dy, ids, (vocab, width), -0.7)
        assert torch.equal(em.lookup(dy, ids % n, 3.0), (dy[ids % n].float() * 3.0).to(dtype))


@pytest.mark.parametrize("n", [20000, 300000])
def test_a_row_of_very_many_tokens(em, n):
    """One word nearly everywhere: parts by the thousand; whole numbers, whose float32 sums are exact in any order."""
    ids = torch.full((n,), 17, device=DEV)
    ids[:: 1000] = torch.arange(n // 1000, device=DEV) % 50
    dy = torch.randint(-3, 4, (n, 24), generator=gen(8), device=DEV).float()
    got = em.lookup_backward(dy, ids, (60, 24))
    assert torch.equal(got, torch.zeros(60, 24, device=DEV, dtype=torch.float64).index_add_(0, ids, dy.double()).float())


def test_more_bits_than_two_passes(em):
    """2^25 table rows: three passes of the sort."""
    g = gen(4)
    ids = torch.randint(0, 1 << 25, (3000,), generator=g, device=DEV)
    ids[::3] = 1 << 24
    check_grad(em, torch.randn(3000, 1, generator=g, device=DEV).to(BF16), ids, (1 << 25, 1))


def test_gradient_beyond_32_bits(em):
    """A gradient of more than 2^32 bytes: rows at its end, and clean rows at its start."""
    vocab, width = 600000, 4096
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device=DEV)
    dy = torch.randn(4, width, generator=gen(), device=DEV).to(BF16)
    grad = em.lookup_backward(dy, ids, (vocab, width))
    assert torch.equal(grad[vocab - 1], (dy[0].float() + dy[3].float()).to(BF16)) and torch.equal(grad[vocab - 2], dy[2])
    assert torch.equal(grad[0], dy[1]) and not grad[1:vocab - 2].any()
    assert torch.equal(em.lookup(grad, ids[:1])[0], grad[vocab - 1])


def test_infinities_stay_in_their_rows(em):
    dy = torch.ones(40, 16, dtype=BF16, device=DEV)
    ids = torch.arange(40, device=DEV) % 5
    want = em.lookup_backward(dy, ids, (9, 16))
    dy[3::5] = float("nan")
    got = em.lookup_backward(dy, ids, (9, 16))
    assert torch.isnan(got[3]).all() and torch.equal(got[[0, 1, 2, 4, 5, 6, 7, 8]], want[[0, 1, 2, 4, 5, 6, 7, 8]])


def test_autograd_strides_and_differences(em):
    """The forward is linear in the table: with small whole numbers a change of one value changes the output by the gradient times it."""
    g = gen(6)
    table = torch.randint(-3, 4, (3, 20, 6), generator=g, device=DEV).to(F32)
    ids = torch.randint(0, 20, (4, 9), generator=g, device=DEV).t()  # strided
    index = torch.tensor([0, 2, 1, 0, 2, 1, 1, 0, 2], device=DEV)
    scale = torch.tensor([2.0, 0.5, 4.0], device=DEV)
    dy = torch.randint(-3, 4, (9, 4, 6), generator=g, device=DEV).to(F32)
    leaf = table.clone().requires_grad_()
    out = em.embed(leaf, ids, scale, adapter_indices=index)
    out.backward(dy.transpose(0, 1).contiguous().transpose(0, 1))
    base = em.lookup(table, ids, scale, adapter_indices=index)
    assert torch.equal(out, base)
    for a, v, c in ((0, int(ids[0, 0]), 0), (2, int(ids[1, 3]), 5), (1, 19, 2)):
        moved = table.clone()
        moved[a, v, c] += 1
        assert float(((em.lookup(moved, ids, scale, adapter_indices=index) - base) * dy).sum()) == float(leaf.grad[a, v, c])
    view = torch.randn(21 * 16 + 1, generator=g, device=DEV).to(BF16)[1:].view(21, 16)  # 2 bytes past 16
    assert torch.equal(em.lookup(view, ids), view[ids])
    check_grad(em, torch.randn(36 * 16 + 1, generator=g, device=DEV).to(BF16)[1:].view(9, 4, 16), ids, (21, 16))


@pytest.mark.parametrize("n", [500, 70000])
def test_graph_replays(em, n):
    g = gen(7)
    ids = torch.randint(0, 3000, (n,), generator=g, device=DEV)
    dy = torch.randn(n, 32, generator=g, device=DEV).to(BF16)
    fresh = [torch.randint(0, 50 * (i + 1), (n,), generator=g, device=DEV) for i in range(3)]
    em.lookup_backward(dy, ids, (3000, 32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = em.lookup_backward(dy, ids, (3000, 32))
        rows = em.lookup(grad, ids, 0.5)
    for f in fresh:
        ids.copy_(f)
        graph.replay()
        eager = em.lookup_backward(dy, ids, (3000, 32))
        torch.cuda.synchronize()
        assert torch.equal(grad, eager) and torch.equal(rows, em.lookup(eager, ids, 0.5))


def test_the_most_tokens(em):
    """2^20 tokens; the last rows of the output lie 4.3 GB behind the first."""
    n, vocab = 1 << 20, 5000
    g = gen(9)
    table = torch.randn(vocab, 2056, generator=g, device=DEV).to(BF16)
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    out = em.lookup(table, ids)
    for r in (slice(0, 10), slice(n // 2, n // 2 + 10), slice(n - 10, n)):
        assert torch.equal(out[r], table[ids[r]])
    del out
    dy = torch.randint(-3, 4, (n, 9), generator=g, device=DEV).float()
    want = torch.zeros(vocab, 9, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
    assert torch.equal(em.lookup_backward(dy, ids, (vocab, 9)), want.float())
    with pytest.raises(ValueError, match="at most"):
        em.lookup(table, torch.zeros(n + 1, dtype=torch.int64, device=DEV))


def test_the_widest_rows(em):
    g = gen(10)
    ids = torch.tensor([3, 0, 3, 2, 3], device=DEV)
    for width in (65536, 65535):
        dy = torch.randint(-3, 4, (5, width), generator=g, device=DEV).to(BF16)
        want = torch.zeros(5, width, device=DEV).index_add_(0, ids, dy.float())
        grad = em.lookup_backward(dy, ids, (5, width))
        assert torch.equal(grad.float(), want) and torch.equal(em.lookup(grad, ids).float(), want[ids])


@pytest.mark.parametrize("width,n", [(65536, (1 << 18) + 5), (16384, (1 << 16) + 3), (16384, 1 << 16), (65535, 20000)])
def test_more_units_than_an_axis_of_a_launch(em, width, n):
    """2^28 units (a plane of workgroups) and 2^32 (the threads of an axis) and more: 69 GB of float32 rows, compared 1 GB at a time."""
    print(f"[case] {n} x {width}", flush=True)
    g = gen(11)
    table = torch.randn(3, width, generator=g, device=DEV)
    ids = torch.randint(0, 3, (n,), generator=g, device=DEV)
    out = em.lookup(table, ids)
    step = (1 << 28) // width
    for r in range(0, n, step):
        assert torch.equal(out[r:r + step], table[ids[r:r + step]]), r
