"""Norm and clipping of a group of tensors against 64 bits."""
import numpy as np
import pytest

from ulmblas_amd import blas

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"torch.float32": 2.0 ** -24, "torch.bfloat16": 2.0 ** -8}


def make(sizes, types, seed, scale=1.0, off=0):
    """Tensors that start `off` elements into 16 bytes, with other values around them."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = {"s": torch.float32, "b": torch.bfloat16}[types[i % len(types)]]
        flat = torch.full((n + off + 16,), 1e30, dtype=dt, device="cuda")
        x = flat[off:off + n]
        x.copy_(torch.randn(n, generator=gen, device="cuda") * scale * 10.0 ** -(i % 3))
        out.append(x)
    return out


def norm64(tensors):
    return float(sum((x.double() ** 2).sum() for x in tensors)) ** 0.5 if tensors else 0.0


def around(x):
    """Every element of x's memory that is not x's."""
    import torch
    whole = torch.empty(0, dtype=x.dtype, device="cuda").set_(x.untyped_storage())
    return torch.cat([whole[:x.storage_offset()], whole[x.storage_offset() + x.numel():]])


SIZES = [[1], [0, 5, 0], [7, 8, 9], [2047, 2048, 2049], [1, 100000, 3, 0, 70001], [5] * 128, [11] * 129, [300] * 400,
         [3000001, 17]]


@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
@pytest.mark.parametrize("types", ["s", "b", "sb"])
@pytest.mark.parametrize("off", [0, 1, 7])
def test_norm_and_clip(sizes, types, off):
    import torch
    group = make(sizes, types, sum(sizes) + off, off=off)
    before = [x.clone() for x in group]
    work = torch.full((blas.gnrm2_worksize(group),), 0xff, dtype=torch.uint8, device="cuda")
    norm = torch.full((2,), 7.5, device="cuda")
    blas.gpu_gnrm2(group, norm, work=work)
    n64 = norm64(before)
    # squares exact in 64 bits, sums and root off by far less than one rounding to 32 bits
    assert abs(float(norm[0]) - n64) <= 1.01 * U * n64 and float(norm[1]) == 7.5
    for largest in (0.25 * n64, 0.0, 2.0 * n64 + 1.0, float("inf")):
        out = make(sizes, types, 1, off=(off * 3) % 8)
        blas.gpu_gclip(group, norm, largest, out=out)
        torch.cuda.synchronize()
        for x, b, y in zip(group, before, out):
            assert torch.equal(x, b)
            want = b.double() * min(1.0, largest / float(norm[0]))
            # the factor and the product are rounded, then the result to its type
            tol = (HALF[str(b.dtype)] + 3 * U) * want.abs() + 2.0 ** -133
            assert ((y.double() - want).abs() <= tol).all()
            if largest > n64:
                assert torch.equal(x, y)
            assert (around(y) == torch.tensor(1e30, dtype=y.dtype, device="cuda")).all()
    # in place, the same bits as beside
    out = [torch.empty_like(x) for x in group]
    blas.gpu_gclip(group, norm, 0.25 * n64, out=out)
    blas.gpu_gclip(group, norm, 0.25 * n64)
    torch.cuda.synchronize()
    for x, y in zip(group, out):
        assert torch.equal(x, y)
        assert (around(x) == torch.tensor(1e30, dtype=x.dtype, device="cuda")).all()


def test_empty_group():
    import torch
    norm = blas.gpu_gnrm2([])
    assert float(norm) == 0.0
    assert blas.gpu_gclip([], norm, 1.0).tensors == []
    assert float(blas.gpu_gnrm2([torch.empty(0, device="cuda")])) == 0.0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_range(dtype):
    """Squares that neither fp32 nor its smallest numbers hold."""
    import torch
    dt = getattr(torch, dtype)
    for v in (2.0 ** 120, 2.0 ** -120, 2.0 ** -130):
        x = torch.full((1000,), v, dtype=dt, device="cuda")
        n = float(blas.gpu_gnrm2([x]))
        assert abs(n - v * 1000 ** 0.5) <= 1.01 * U * n + 2.0 ** -150
    big = torch.full((4,), torch.finfo(dt).max, dtype=dt, device="cuda")
    assert float(blas.gpu_gnrm2([big])) == float("inf")      # twice the largest number


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_that_are_no_numbers(value, dtype):
    """They show in the norm, and clipping by such a norm changes nothing."""
    import torch
    x = torch.randn(5000, device="cuda").to(getattr(torch, dtype))
    x[4321] = value
    before = x.clone()
    norm = blas.gpu_gnrm2([x])
    n = float(norm)
    assert np.isnan(n) if np.isnan(value) else n == float("inf")
    out = torch.zeros_like(x)
    blas.gpu_gclip([x], norm, 1.0, out=[out])
    blas.gpu_gclip([x], norm, 1.0)
    assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(before))
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(before))


def test_long_tensor_past_31_bits():
    """Element indexes past 2^31."""
    import torch
    n = (1 << 31) + 12345
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-1] = 3.0
    x[5] = 4.0
    norm = blas.gpu_gnrm2([x])
    assert float(norm) == 5.0
    blas.gpu_gclip([x], norm, 2.5)
    assert float(x[-1]) == 1.5 and float(x[5]) == 2.0 and int((x != 0).sum()) == 2


def test_streams_and_determinism():
    import torch
    group = make([100003] * 50, "sb", 3)
    want = float(blas.gpu_gnrm2(group))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        norm = blas.gpu_gnrm2(group, stream=side.cuda_stream)
        side.synchronize()
        assert float(norm) == want


def test_outputs_of_other_kinds_are_refused():
    import torch
    x, y = torch.ones(8, device="cuda"), torch.ones(9, device="cuda")
    norm = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        blas.gpu_gclip([x], norm, 1.0, out=[y])
    with pytest.raises(ValueError):
        blas.gpu_gclip([x], norm, 1.0, out=[y[:8].bfloat16()])
    with pytest.raises(blas.GpuError):
        blas.gpu_gclip([x], norm, -1.0)
    with pytest.raises(ValueError):
        blas.gpu_gnrm2([x], work=torch.empty(8, dtype=torch.uint8, device="cuda"))


def test_overlapping_tensors_are_not_scaled():
    """A tensor that is in the group twice would be scaled twice, or by what the other one left."""
    import torch
    flat, norm = torch.arange(64, device="cuda", dtype=torch.float32), torch.ones(1, device="cuda")
    a, b, c = flat[:32], flat[31:48], flat[48:]
    for tensors in ([a, a], [a, c, b], [flat, b[:0], c]):
        group = blas.TensorGroup(tensors)
        for _ in range(2):
            with pytest.raises(blas.GpuError, match="overlaps"):
                blas.gpu_gclip(group, norm, 0.5)
    for tensors, out in (([a, c], [c.new_empty(32), a[:16]]), ([a, c], [flat[16:48], c]), ([a[:16], c], [b[:16], b[1:17]])):
        with pytest.raises(blas.GpuError, match="overlaps"):
            blas.gpu_gclip(tensors, norm, 0.5, out=out)
    assert (flat.cpu() == torch.arange(64)).all()
    # the norm counts a tensor as often as it is named; neighbours are fine, and so are tensors of no length inside others
    assert abs(float(blas.gpu_gnrm2([c, c])) - float(c.double().norm()) * 2 ** 0.5) < 1e-3
    blas.gpu_gclip([a, flat[32:48], c, flat[40:40]], norm, 0.5)
    assert (flat.cpu() == torch.arange(64) * 0.5).all()


def test_a_norm_beside_and_inside_the_tensors():
    """In a tensor that is read only, or next to one that is written, the norm may lie; inside one that is written not."""
    import torch
    flat = torch.full((40,), 2.0, device="cuda")
    out = torch.empty(39, device="cuda")
    a, norm = flat[:39], flat[39:]
    blas.gpu_gnrm2([a], norm)
    n = float(norm)
    assert abs(n - 2 * 39 ** 0.5) <= 1.01 * U * n
    blas.gpu_gclip([a], norm, 0.5 * n)              # next to it
    assert (a == 1.0).all() and float(norm) == n
    blas.gpu_gclip([flat[1:]], norm, 0.5 * n, out=[out])
    assert (out[:38] == 0.5).all() and float(out[38]) == 0.5 * n and float(norm) == n
    for tensors in ([flat], [flat[1:]], [a[:5], flat[39:]]):
        with pytest.raises(blas.GpuError, match="norm"):
            blas.gpu_gclip(tensors, norm, 0.5 * n)
    assert (a == 1.0).all() and float(norm) == n


def test_a_workspace_beside_and_inside_the_tensors():
    import torch
    size = blas.gnrm2_worksize([None])
    flat = torch.full((size // 4 + 200,), 1.0, device="cuda")
    a = flat[:100]
    assert float(blas.gpu_gnrm2([a], work=flat[100:])) == 10.0
    assert (a == 1.0).all() and (flat[100 + size // 4:] == 1.0).all()
    for work in (flat, flat[98:]):
        with pytest.raises(blas.GpuError, match="workspace overlaps"):
            blas.gpu_gnrm2([a], work=work)
    assert (a == 1.0).all()


def test_tensors_whose_memory_was_replaced():
    import torch
    x, y = torch.full((100,), 3.0, device="cuda"), torch.full((100,), 4.0, device="cuda")
    group = blas.TensorGroup([x, y])
    assert float(blas.gpu_gnrm2(group)) == 50.0
    old = x.data
    x.data = torch.zeros(100, device="cuda")
    norm = torch.full((1,), 50.0, device="cuda")
    with pytest.raises(ValueError, match="tensor 0 was replaced"):
        blas.gpu_gnrm2(group)
    with pytest.raises(ValueError, match="tensor 0 was replaced"):
        blas.gpu_gclip(group, norm, 25.0)
    assert (old == 3.0).all() and (y == 4.0).all()
    assert float(blas.gpu_gnrm2(blas.TensorGroup([x, y]))) == 40.0
    x.data = old                        # back again
    blas.gpu_gclip(group, norm, 25.0)
    assert (x == 1.5).all() and (y == 2.0).all()
