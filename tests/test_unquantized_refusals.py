"""What the bf16 grouped products, the embedding rows and the gradient clipping refuse, on the CPU: the C calls with addresses that are
never read, the Python entry points with CPU tensors."""

import ctypes
import sys
import threading
import time

import pytest
import torch

from __graft_entry__ import load_package

A = 0x100000  # never dereferenced: validation fails first
STEP = 0x10000000


@pytest.fixture(scope="module")
def native():
    native = load_package()._native
    if not native.LIB_PATH.exists():
        pytest.skip("libmi355_w8a8.so not built (run __graft_entry__.build())")
    return native


def fill(struct, **kw):
    p = struct()
    p.struct_size = ctypes.sizeof(struct)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), -8), (dict(flags=1), -2), (dict(flags=12), -2), (dict(m=0), -2), (dict(n_groups=0), -2), (dict(k=12), -7), (dict(n=4), -7),
    (dict(k=65544), -7), (dict(n_groups=1025), -7), (dict(m=(1 << 20) + 1), -7), (dict(x=None), -1), (dict(weight=None), -1),
    (dict(group_sizes=None), -1), (dict(out=None), -1), (dict(x=A + 8), -3), (dict(weight=A + STEP + 2), -3),
    (dict(group_sizes=A + 2), -3), (dict(out=A + 16), -4), (dict(out=A + STEP + 1024), -4)])
def test_grouped_call(native, change, status):
    p = fill(native.Bf16GroupedProblem, **{**dict(m=16, k=64, n=32, n_groups=4, x=A, weight=A + STEP, group_sizes=A + 2 * STEP,
                                                  out=A + 3 * STEP), **change})
    assert native.load().mi355_w8a8_bf16_grouped_v1(ctypes.byref(p), None) == status
    assert native.load().mi355_w8a8_bf16_grouped_v1(None, None) == -1


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), -8), (dict(flags=2), -2), (dict(n=0), -2), (dict(k=4), -7), (dict(dy=None), -1), (dict(dx=None, dw=None), -1),
    (dict(weight=None), -1), (dict(x=None), -1), (dict(dx=A + 3 * STEP + 4), -3), (dict(dw=A + STEP), -4), (dict(dx=A), -4),
    (dict(dx=A + 3 * STEP, dw=A + 3 * STEP + 512), -4), (dict(dw=A + 2 * STEP), -4)])
def test_grouped_backward_call(native, change, status):
    p = fill(native.Bf16GroupedBwdProblem, **{**dict(m=16, k=64, n=32, n_groups=4, x=A, dy=A + STEP, weight=A + 2 * STEP,
                                                     dx=A + 3 * STEP, dw=A + 4 * STEP, group_sizes=A + 5 * STEP), **change})
    assert native.load().mi355_w8a8_bf16_grouped_bwd_v1(ctypes.byref(p), None) == status


def test_grouped_workspace(native):
    lib = native.load()
    sizes = dict(m=1, k=4096, n=4096, n_groups=8)
    need = lib.mi355_w8a8_bf16_grouped_workspace_bytes(1, 4096, 4096, 8, 0)
    back = lib.mi355_w8a8_bf16_grouped_bwd_workspace_bytes(1, 4096, 4096, 8, 0, 1, 1)
    assert need >= 2 * 4096 * 4 and back >= 2 * 4096 * 4
    assert lib.mi355_w8a8_bf16_grouped_bwd_workspace_bytes(1, 4096, 4096, 8, 0, 0, 0) == 0 and lib.mi355_w8a8_bf16_grouped_workspace_bytes(1, 12, 8, 8, 0) == 0
    W = A + 9 * STEP
    for change, status in ((dict(), -5), (dict(workspace=W, workspace_bytes=need - 1), -5), (dict(workspace=W + 64, workspace_bytes=need), -3),
                           (dict(workspace=A + 3 * STEP, workspace_bytes=need), -4), (dict(workspace=A + STEP, workspace_bytes=need), -4)):
        p = fill(native.Bf16GroupedProblem, **{**sizes, **dict(x=A, weight=A + STEP, group_sizes=A + 8 * STEP, out=A + 3 * STEP), **change})
        assert lib.mi355_w8a8_bf16_grouped_v1(ctypes.byref(p), None) == status, change
    for change, status in ((dict(), -5), (dict(workspace=W, workspace_bytes=back - 1), -5), (dict(workspace=W + 64, workspace_bytes=back), -3),
                           (dict(workspace=A + 5 * STEP, workspace_bytes=back), -4), (dict(workspace=A + 3 * STEP, workspace_bytes=back), -4)):
        p = fill(native.Bf16GroupedBwdProblem, **{**sizes, **dict(x=A, dy=A + STEP, weight=A + 3 * STEP, dx=A + 2 * STEP, dw=A + 5 * STEP,
                                                                  group_sizes=A + 8 * STEP), **change})
        assert lib.mi355_w8a8_bf16_grouped_bwd_v1(ctypes.byref(p), None) == status, change


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=8), -8), (dict(flags=4), -2), (dict(n_tokens=0), -2), (dict(vocab=0), -2), (dict(width=0), -2),
    (dict(n_tokens=(1 << 20) + 1), -7), (dict(width=65537), -7), (dict(vocab=(1 << 30) + 1), -7), (dict(n_adapters=2), -1),
    (dict(n_adapters=1 << 22, vocab=1 << 22, adapter_indices=A + 2 * STEP), -7), (dict(adapter_indices=A), -2), (dict(scales=A), -2),
    (dict(ids=None), -1), (dict(ids=A + 2), -3), (dict(flags=2, ids=A + 4), -3), (dict(out=None), -1)])
def test_embedding_calls(native, change, status):
    base = dict(n_tokens=8, vocab=100, width=24, ids=A, table=A + STEP, d_out=A + STEP, out=A + 3 * STEP, workspace=A + 4 * STEP,
                workspace_bytes=1 << 20)
    lib = native.load()
    for fn in (lib.mi355_w8a8_embedding_v1, lib.mi355_w8a8_embedding_bwd_v1):
        assert fn(ctypes.byref(fill(native.EmbeddingProblem, **{**base, **change})), None) == status
    fwd = lambda **kw: lib.mi355_w8a8_embedding_v1(ctypes.byref(fill(native.EmbeddingProblem, **{**base, **kw})), None)
    bwd = lambda **kw: lib.mi355_w8a8_embedding_bwd_v1(ctypes.byref(fill(native.EmbeddingProblem, **{**base, **kw})), None)
    assert fwd(table=None) == -1 and bwd(d_out=None) == -1
    assert fwd(out=A + STEP + 64) == -4 and bwd(out=A + STEP) == -4 and fwd(out=A) == -4
    assert fwd(table=A + STEP + 1) == -3 and bwd(out=A + 3 * STEP + 8) == -3
    assert bwd(workspace=None) == -5 and bwd(workspace_bytes=64) == -5 and bwd(workspace=A + 4 * STEP + 16) == -3
    assert bwd(workspace=A + 3 * STEP) == -4
    assert lib.mi355_w8a8_embedding_bwd_workspace_bytes(0, 100, 8, 0, 0) == 0
    assert lib.mi355_w8a8_embedding_bwd_workspace_bytes(8, 100, 8, 0, 0) % 256 == 0


def test_gradient_calls(native):
    lib = native.load()

    def clip(tensors, adapters=2, limits=A, norms=A + 64, ws=A + 5 * STEP, ws_bytes=1 << 20, n=None, flags=0):
        table = (native.GradTensor * max(1, len(tensors)))(*[native.GradTensor(*t) for t in tensors])
        return lib.mi355_w8a8_grad_clip_v1(table, len(tensors) if n is None else n, adapters, limits, norms, ws, ws_bytes, flags, None)

    good = (A + STEP, A + 2 * STEP, 100, 0, 0)
    assert lib.mi355_w8a8_grad_clip_v1(None, 1, 1, A, A, A, 1, 0, None) == -1
    assert clip([]) == -2 and clip([good], adapters=0) == -2 and clip([good], adapters=65536) == -7
    assert clip([good], flags=2) == -2
    assert clip([good], limits=None) == -1 and clip([good], norms=None) == -1
    assert clip([(None, A, 100, 0, 0)]) == -1 and clip([(A + STEP, None, 100, 0, 0)]) == -1
    assert clip([(A + STEP, A + 2 * STEP, 100, 2, 0)]) == -2 and clip([(A + STEP, A + 2 * STEP, 100, 0, 1)]) == -2
    assert clip([(A + STEP + 1, A + 2 * STEP, 100, 0, 0)]) == -3 and clip([(A + STEP + 2, A + 2 * STEP, 100, 1, 0)]) == -3
    assert clip([(A + STEP, A + STEP + 16, 100, 0, 0)]) == -4 and clip([good], norms=A + STEP) == -4 and clip([good], limits=A + 2 * STEP) == -4
    assert clip([good], ws=None) == -5 and clip([good], ws_bytes=4) == -5 and clip([good], ws=A + 5 * STEP + 8) == -3
    assert clip([good], ws=A + STEP) == -4 and clip([(A + STEP, A + 2 * STEP, 1 << 40, 0, 0)]) == -7
    assert lib.mi355_w8a8_grad_norm_v1((native.GradTensor * 1)(native.GradTensor(*good)), 1, 1, None, A, 1 << 20, 0, None) == -1


def test_python_grouped(native):
    gl = load_package().bf16_grouped_linear
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    sizes = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="BF16"):
        gl.grouped_matmul(torch.zeros(4, 8), bf(2, 8, 8), sizes)
    with pytest.raises(RuntimeError, match="GPU"):
        gl.grouped_matmul(bf(4, 8), bf(2, 8, 8), sizes)
    with pytest.raises(TypeError, match="dw_dtype"):
        gl.grouped_matmul_backward(bf(4, 8), bf(4, 8), bf(2, 8, 8), sizes, dw_dtype=torch.float16)
    with pytest.raises(ValueError, match="needs"):
        gl.grouped_matmul_backward(None, bf(4, 8), bf(2, 8, 8), sizes)
    geometry = lambda x, w, s: gl._geometry(x, "x", 1, w.shape, s)
    for x, w, s in ((bf(4, 8), bf(8, 8), sizes), (bf(4, 16), bf(2, 8, 8), sizes), (bf(0, 8), bf(2, 8, 8), sizes), (bf(4, 2, 8), bf(2, 8, 8), sizes),
                    (bf(4, 8), bf(2, 8, 8), torch.zeros(3, dtype=torch.int32)), (bf(4, 12), bf(2, 12, 8), sizes), (bf(4, 8), bf(2, 8, 20), sizes),
                    (bf(4, 8), bf(1025, 8, 8), torch.zeros(1025, dtype=torch.int32))):
        with pytest.raises(ValueError):
            geometry(x, w, s)
    with pytest.raises(TypeError, match="integers"):
        geometry(bf(4, 8), bf(2, 8, 8), torch.zeros(2))


def test_python_embedding(native):
    em = load_package().embedding
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        em.lookup(torch.zeros(4, 8), ids)
    with pytest.raises(RuntimeError, match="GPU"):
        em.lookup_backward(torch.zeros(3, 8), ids, (4, 8))
    dev = torch.device("cpu")

    def problem(ids=ids, shape=(4, 8), scale=None, index=None, dtype=torch.bfloat16):
        return em._problem(ids, shape, scale, index, dtype, dev)

    with pytest.raises(TypeError, match="FP32"):
        problem(dtype=torch.float16)
    with pytest.raises(TypeError, match="INT"):
        problem(ids=torch.zeros(3))
    with pytest.raises(RuntimeError, match="GPU"):
        problem()
    leaf = torch.ones(2, requires_grad=True)
    with pytest.raises(ValueError, match="constant"):
        em.embed(torch.zeros(2, 4, 8), ids, leaf, adapter_indices=ids)


def test_python_clipping(native):
    gc = load_package().grad_clip
    with pytest.raises(ValueError, match="at least one"):
        gc.grad_norm([])
    with pytest.raises(TypeError, match="BF16"):
        gc.grad_norm([torch.zeros(3, dtype=torch.float16)])
    with pytest.raises(RuntimeError, match="GPU"):
        gc.grad_norm([torch.zeros(3)])
    with pytest.raises(TypeError, match="bool"):
        gc.clip_grad_norm([torch.zeros(3)], 1.0, per_adapter=1)


def test_capture_beside_a_living_graph(native, monkeypatch):
    """The rule alone, with streams and captures that are only claimed."""
    from skyrl_tx_rocm_amd.kernels.rocm import bf16_grouped_linear as gl
    stream, capturing = [1], [False]
    monkeypatch.setattr(gl, "_stream_ptr", lambda device: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    leaf, other = torch.zeros(2, requires_grad=True), torch.zeros(2, requires_grad=True)
    eager = gl.note_leaves(leaf, leaf * 2, torch.zeros(2))
    assert len(eager) == 1
    gl.check_capture(eager)
    stream[0], capturing[0] = 2, True
    gl.check_capture(gl.note_leaves(other, leaf * 2))
    mine = gl.note_leaves(leaf)
    with pytest.raises(RuntimeError, match="lives"):
        gl.check_capture(mine)
    del eager
    gl.check_capture(mine)
    capturing[0] = False
    gl.check_capture(mine)


@pytest.mark.parametrize("flags", [1, 2, 5, 12, 32, -1, 1 << 32, 1 << 40])
def test_flags_that_are_no_tiles(native, flags):
    """Above all the C call's flag of a float32 dw (1): beside a bf16 dw its stores would go past the tensor's end."""
    gl = load_package().bf16_grouped_linear
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    sizes = torch.zeros(2, dtype=torch.int32)
    assert native.FLAG_BF16_GROUPED_DW_F32 == 1
    with pytest.raises(ValueError, match="flags"):
        gl.grouped_matmul(bf(4, 8), bf(2, 8, 8), sizes, flags=flags)
    for dtype in (torch.bfloat16, torch.float32):
        with pytest.raises(ValueError, match="flags"):
            gl.grouped_matmul_backward(bf(4, 8), bf(4, 8), bf(2, 8, 8), sizes, dw_dtype=dtype, flags=flags)
    for tile in (0, 4, 8, 16):  # (these go on, to the next check)
        with pytest.raises(RuntimeError, match="GPU"):
            gl.grouped_matmul(bf(4, 8), bf(2, 8, 8), sizes, flags=tile)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64])
def test_whole_numbers_of_any_width(native, monkeypatch, dtype):
    """Sizes and adapter indices keep their values where there are more rows or adapters than their type can hold."""
    from skyrl_tx_rocm_amd.kernels.rocm import bf16_grouped_linear as gl, embedding as em
    sizes = gl._geometry(torch.zeros(40000, 8, dtype=torch.bfloat16), "x", 1, (3, 8, 8), torch.tensor([100, 0, 27], dtype=dtype))[-1]
    assert sizes.dtype == torch.int32 and sizes.tolist() == [100, 0, 27]
    monkeypatch.setattr(em, "_require_cuda", lambda t, name: None)
    ids = torch.zeros(3, dtype=torch.int64)
    for adapters, given in ((2, [0, 1, 1]), (40000, [0, 127, 3])):
        _, (_, index, _) = em._problem(ids, (adapters, 4, 8), None, torch.tensor(given, dtype=dtype), torch.bfloat16, ids.device)
        assert index.dtype == torch.int32 and index.tolist() == given
    if dtype.is_signed:
        assert gl._geometry(torch.zeros(40000, 8, dtype=torch.bfloat16), "x", 1, (2, 8, 8), torch.tensor([-7, 3], dtype=dtype))[-1].tolist()[0] <= 0
        assert int(em._problem(ids, (2, 4, 8), None, torch.tensor([-1, -128, 1], dtype=dtype), torch.bfloat16, ids.device)[1][1][:2].max()) < 0
    if dtype in (torch.int64, torch.uint32):  # what int32 cannot hold is out of range, not another number
        assert gl._geometry(torch.zeros(40000, 8, dtype=torch.bfloat16), "x", 1, (2, 8, 8), torch.tensor([2 ** 32 - 1, 3], dtype=dtype))[-1].tolist() == [40000, 3]
        assert em._problem(ids, (2, 4, 8), None, torch.tensor([2 ** 32 - 1, 2 ** 31, 1], dtype=dtype), torch.bfloat16, ids.device)[1][1].tolist() == [2, 2, 1]


def test_what_are_no_whole_numbers(native, monkeypatch):
    from skyrl_tx_rocm_amd.kernels.rocm import bf16_grouped_linear as gl, embedding as em
    monkeypatch.setattr(em, "_require_cuda", lambda t, name: None)
    ids = torch.zeros(2, dtype=torch.int64)
    for dtype in (torch.float32, torch.bool, torch.complex64, torch.uint64):
        with pytest.raises(TypeError, match="integers"):
            gl._geometry(torch.zeros(4, 8, dtype=torch.bfloat16), "x", 1, (2, 8, 8), torch.zeros(2, dtype=dtype))
        with pytest.raises(TypeError, match="integers"):
            em._problem(ids, (2, 4, 8), None, torch.zeros(2, dtype=dtype), torch.bfloat16, ids.device)


def test_forward_mode_tangents(native):
    """No tangent is dropped: the calls that autograd may differentiate say that they have none to give, whether a gradient is required or not."""
    from torch.autograd import forward_ad
    pkg = load_package()
    gl, em = pkg.bf16_grouped_linear, pkg.embedding
    x, w, sizes = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    ids = torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        for required in (False, True):
            dual = lambda t: forward_ad.make_dual(t.clone().requires_grad_(required), torch.ones_like(t))
            for call in (lambda: gl.bf16_grouped_linear(dual(x), w, sizes), lambda: gl.bf16_grouped_linear(x, dual(w), sizes), lambda: em.embed(dual(x), ids),
                         lambda: em.embed(dual(w), ids, adapter_indices=ids)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            em.embed(w, ids, forward_ad.make_dual(torch.ones(2), torch.ones(2)), adapter_indices=ids)
        with pytest.raises(RuntimeError, match="GPU"):  # a level alone is no tangent
            gl.bf16_grouped_linear(x, w, sizes)
    with pytest.raises(RuntimeError, match="GPU"):
        gl.bf16_grouped_linear(x, w, sizes)


def test_captures_beside_forwards_of_other_threads(native, monkeypatch):
    """The rule is looked at while other threads record uses of their own leaves: neither waits for nor disturbs the other."""
    from skyrl_tx_rocm_amd.kernels.rocm import bf16_grouped_linear as gl
    monkeypatch.setattr(gl, "_stream_ptr", lambda device: 1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    kept, stop, failed = [], threading.Event(), []
    mine = gl.note_leaves(torch.zeros(2, requires_grad=True))

    def forwards():
        while not stop.is_set():
            kept.append(gl.note_leaves(*[torch.zeros(1, requires_grad=True) for _ in range(8)]))

    workers = [threading.Thread(target=forwards) for _ in range(4)]
    try:
        for w in workers:
            w.start()
        end = time.monotonic() + 3.0
        while time.monotonic() < end and not failed:
            try:
                gl.check_capture(mine)
            except RuntimeError as e:
                failed.append(e)
    finally:
        stop.set()
        for w in workers:
            w.join()
        sys.setswitchinterval(interval)
    assert not failed


@pytest.mark.parametrize("rows,k,n,groups,tiles", [
    (4051, 128, 120, 22, (16, 16)), (886, 168, 736, 13, (16, 16)), (1003, 712, 1096, 13, (8, 8)), (4096, 1024, 1024, 8, (8, 8)), (300, 64, 280, 28, (16, 16)),
    (8000, 1576, 1744, 25, (8, 8)), (1, 8, 8, 1, (16, 16)), (70, 40, 136, 1024, (16, 16)),
    (560, 1944, 2072, 115, (0, 0)), (32768, 768, 2048, 128, (0, 0)),  # bytes bound both
    (9000, 8, 520, 1, (0, 0)), (1, 4096, 4096, 8, (0, 0)),            # parts of a contraction
    (1, 12, 8, 1, (0, 0))])
def test_sizes_whose_gradients_share_a_launch(native, rows, k, n, groups, tiles):
    """The sizes that test_both_gradients_and_each of the GPU tests takes for this, and others; a bf16 dw and a float32 one."""
    joint = native.load().mi355_w8a8_bf16_grouped_bwd_joint_tile
    assert tuple(joint(rows, k, n, groups, f32) for f32 in (0, native.FLAG_BF16_GROUPED_DW_F32)) == tiles
    if k % 8 == 0:
        assert [joint(rows, k, n, groups, f) for f in (4, 8, 16)] == [4, 8, 16]


def test_scales_that_float32_cannot_hold(native, monkeypatch):
    """The product is float32: a larger scale would be an infinity there, also where the product itself could be held."""
    from skyrl_tx_rocm_amd.kernels.rocm import embedding as em
    monkeypatch.setattr(em, "_require_cuda", lambda t, name: None)
    ids = torch.zeros(3, dtype=torch.int64)
    of = lambda scale: em._problem(ids, (4, 8), scale, None, torch.bfloat16, ids.device)[0].scale
    for bad in (float("inf"), float("nan"), 1e39, -3.5e38, 10 ** 40):
        with pytest.raises(ValueError, match="finite"):
            of(bad)
    assert of(None) == 1.0 and of(-2) == -2.0 and of(torch.finfo(torch.float32).max) == torch.finfo(torch.float32).max and of(1e-50) == 0.0
