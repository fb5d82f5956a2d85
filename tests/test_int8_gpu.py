"""Products of weights in 8-bit integers against the same sums in 64 bits, and what they refuse."""

import pytest
import torch

from qwen3_runtime_amd.ops import Int8Weight

DEV = "cuda:0"
gpu = pytest.mark.gpu


def rnd(*shape, seed=0, dtype=torch.float32, device=DEV):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def codes_of(x):
    """Codes and scales of rows by the definition: 127 / the largest magnitude, and the product with it, in float32."""
    most = x.float().abs().amax(-1)
    top = torch.full_like(most, 127)  # a tensor: a quotient with a number is a product with its reciprocal
    by = torch.where(most < 2.0 ** -100, 0.0, top / most)
    return (x.float() * by[:, None]).round(), most / top


def product(x, w):
    q, s = codes_of(x)
    return (q.double() @ w.values[:, : w.shape[1]].double().t()) * s.double()[:, None] * w.scale.double()


def ops():
    from qwen3_runtime_amd.ops.hip import HipOps

    return HipOps()


# Sum and scales in float32: the sum of whole numbers is rounded to 24 bits once, two products round once each: 3 * 2^-24. A result in
# bfloat16 is rounded once more, by 2^-8 of it at most.
STEP = {torch.float32: 3.2 * 2.0 ** -24, torch.bfloat16: 2.0 ** -8 * 1.001}


def near(got, want, dtype, what=""):
    off = (got.double() - want).abs() - STEP[dtype] * want.abs()
    assert got.dtype == dtype and float(off.max()) <= 1e-30, f"{what} {float(off.max())}"


ROWS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 48, 49, 64, 65, 130, 257]


@gpu
@pytest.mark.parametrize("k", [1, 7, 128, 136, 1100, 2560, 9728])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_of_rows(k, dtype):
    x = rnd(9, k, seed=k, dtype=dtype)
    x[1] = 0
    x[2] *= 1e-33
    x[3, -1] = -1000
    got, scale = ops().quantize_rows(x)
    q, s = codes_of(x)
    assert got.shape[1] % 128 == 0 and torch.equal(got[:, :k].float(), q) and not got[:, k:].any()
    assert torch.equal(scale, s)


@gpu
@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(5, 1), (16, 128), (96, 272), (333, 1100), (1000, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products(m, n, k, dtype):
    x, w = rnd(m, k, seed=m, dtype=dtype), Int8Weight.quantize(rnd(n, k, seed=n))
    near(ops().linear(x, w), product(x, w), dtype)
    near(ops().linear(x, w, out_f32=True), product(x, w), torch.float32)
    near(ops().linear_for_residual(x, w), product(x, w), torch.float32)


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 6144, 2560), (8, 2560, 9728), (16, 2560, 4096), (24, 6144, 4096), (40, 2560, 4096), (64, 1024, 9728), (300, 2560, 9728), (2047, 6144, 2560)])
def test_products_of_a_models_sizes(m, n, k):
    x, w = rnd(m, k, seed=m, dtype=torch.bfloat16), Int8Weight.quantize(rnd(n, k, seed=n))
    near(ops().linear(x, w), product(x, w), torch.bfloat16)


@gpu
@pytest.mark.parametrize("tile", range(14))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n", [304, 301])
def test_every_tile(tile, gated, n, monkeypatch):
    o = ops()
    monkeypatch.setattr(type(o), "choose_tile", staticmethod(lambda *a: (tile, 1)))
    m, k = 270, 650
    x, w = rnd(m, k, seed=1, dtype=torch.bfloat16), Int8Weight.quantize(rnd(2 * n if gated else n, k, seed=2) / 25)
    for dtype in (torch.bfloat16, torch.float32):
        x = x.to(dtype)
        if gated:
            near_gated(o.gated_linear(x, w), x, w, dtype)
        else:
            near(o.linear(x, w), product(x, w), dtype)


def near_gated(got, x, w, dtype, activation="swiglu", limit=0.0):
    """Gate and up values are off by 3 * 2^-24 of themselves; the activation's slope is at most 1.1 and its own
    evaluation off by some 5 * 2^-24 of it, x * sigmoid(x) by |x| times that of the sigmoid's argument: (8 + 2 |gate|) * 2^-24."""
    y = product(x, w)
    g, u = y.chunk(2, -1)
    if activation == "clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        want, per = g * torch.sigmoid(1.702 * g) * u, (12 + 4 * g.abs()) * 2.0 ** -24
    else:
        want, per = g * torch.sigmoid(g) * u, (12 + 4 * g.abs()) * 2.0 ** -24
    off = (got.double() - want).abs() - want.abs() * (per + (2.0 ** -8 * 1.001 if dtype == torch.bfloat16 else 0.0))
    if activation == "clamped":  # up + 1 may cancel: up's own error counts whole
        off -= 4 * 2.0 ** -24 * (g.abs() * (u.abs() + 1))
    assert got.dtype == dtype and float(off.max()) <= 1e-30, float(off.max())


@gpu
@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(5, 3), (64, 128), (333, 1100), (1000, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gated_products(m, n, k, dtype):
    x, w = rnd(m, k, seed=m, dtype=dtype), Int8Weight.quantize(rnd(2 * n, k, seed=n) * k ** -0.5)
    near_gated(ops().gated_linear(x, w), x, w, dtype)
    near_gated(ops().gated_linear(x, w, "clamped", 1.5), x, w, dtype, "clamped", 1.5)


@gpu
@pytest.mark.parametrize("planes", [0, 1, 3])
@pytest.mark.parametrize("m,h,n", [(1, 96, 40), (5, 640, 304), (20, 2560, 301), (70, 1100, 64), (3, 8192, 32), (2, 8320, 32), (2, 102, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_norms_codes_and_their_products(m, h, n, planes, dtype):
    """As the norm and the products behind it, apart; the norm's sums may be made in another order, which moves a code by one here and there (1 / 127 of
    a row's largest element, of h elements)."""
    o = ops()
    delta = None if planes == 0 else rnd(planes, m, h, seed=4) if planes > 1 else rnd(m, h, seed=4, dtype=torch.bfloat16)
    residual, weight, w = rnd(m, h, seed=1), 1 + rnd(h, seed=2) / 10, Int8Weight.quantize(rnd(n, h, seed=3))
    one, other = residual.clone(), residual.clone()
    rows = o.add_rmsnorm_codes(one, delta, weight, 1e-5, dtype)
    plain = o.add_rmsnorm(other, delta, weight, 1e-5, dtype)
    # planes join the stream one after the other, or their sum does
    assert torch.allclose(one, other, rtol=0, atol=1e-5)
    codes, scale = o.quantize_rows(plain)
    if hasattr(rows, "codes"):
        off = (rows.codes.int() - codes.int()).abs()
        assert int(off.max()) <= 1 and float((off > 0).float().mean()) < 2e-3 and torch.allclose(rows.scale, scale, rtol=2 ** -7)
    else:
        assert h % 4 or h > 8192
    for a, b in ((o.linear(rows, w), o.linear(plain, w)), (o.linear_for_residual(rows, w), o.linear_for_residual(plain, w)),
                 (o.gated_linear(rows, w), o.gated_linear(plain, w)) if n % 2 == 0 else (weight, weight)):
        assert a.dtype == b.dtype and float((a - b).double().norm()) <= 0.01 * float(b.double().norm())


@gpu
@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("m,n,k", [(33, 304, 1280), (48, 301, 2560), (70, 1024, 9728), (130, 96, 4100), (600, 256, 2300)])
def test_products_for_the_residual_in_planes(m, n, k, coded):
    """The planes' whole sums meet in float32: each is rounded three times, and their sum once more a plane, all relative to the magnitudes of the planes."""
    from qwen3_runtime_amd.ops.hip import CodedRows, HipOps

    o = HipOps(residual_planes=True)
    x, w = rnd(m, k, seed=m, dtype=torch.bfloat16), Int8Weight.quantize(rnd(n, k, seed=n))
    got = o.linear_for_residual(CodedRows(*o.quantize_rows(x), x.shape, x.dtype) if coded else x, w)
    assert (got.dim() == 3) == (k >= 2048) and got.dtype == torch.float32  # a plane has eight stages of 128 columns or more
    got = got.view(-1, m, n)
    parts = got.shape[0]
    want = product(x, w)
    assert bool(((got.double().sum(0) - want).abs() <= STEP[torch.float32] * got.double().abs().sum(0)).all())
    # the norm behind adds them up, one after the other or their sum: as many roundings as there are planes either way
    if n % 4 == 0:
        ours, again = rnd(m, n, seed=5), rnd(m, n, seed=5)
        o.add_rmsnorm_codes(ours, got, rnd(n, seed=6), 1e-6, torch.bfloat16)
        o.add_rmsnorm(again, got, rnd(n, seed=6), 1e-6, torch.bfloat16)
        assert torch.allclose(ours, again, rtol=0, atol=2 * parts * 2.0 ** -24 * float((got.abs().sum(0) + rnd(m, n, seed=5).abs()).max()))
    # few rows, and a caller that takes no planes, get the whole
    assert o.linear_for_residual(x[:32].contiguous(), w).shape == (32, n)
    assert ops().linear_for_residual(x, w).shape == (m, n)


@gpu
@pytest.mark.parametrize("m", [3, 20, 100])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite_are_nan_and_leave_the_others(m, bad):
    x, w = rnd(m, 640, seed=3, dtype=torch.bfloat16), Int8Weight.quantize(rnd(96, 640, seed=4))
    x[0] = 0
    want = ops().linear(x, w)
    assert not want[0].any()
    x[1, 639] = bad
    got = ops().linear(x, w)
    assert got[1].isnan().all()
    keep = torch.arange(m) != 1
    assert torch.equal(got[keep], want[keep])


@gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(2, 300, 2560), (24, 300, 1100), (300, 512, 1280)])
def test_a_captured_product_is_the_eager_one(m, n, k):
    o = ops()
    x, w = rnd(m, k, seed=1, dtype=torch.bfloat16), Int8Weight.quantize(rnd(n, k, seed=2))
    o.linear(x, w), o.gated_linear(x, w)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, z = o.linear(x, w), o.gated_linear(x, w)
    for seed in range(4):
        x.copy_(rnd(m, k, seed=seed + 7, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, o.linear(x, w)) and torch.equal(z, o.gated_linear(x, w))


@gpu
def test_products_on_another_stream():
    o, s = ops(), torch.cuda.Stream()
    x, w = rnd(40, 640, seed=1, dtype=torch.bfloat16), Int8Weight.quantize(rnd(320, 640, seed=2))
    want = o.linear(x, w)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = o.linear(x, w)
    s.synchronize()
    assert torch.equal(got, want)


@gpu
def test_no_rows_and_refusals_on_the_device():
    from qwen3_runtime_amd.ops import OpsError

    o, w = ops(), Int8Weight.quantize(rnd(30, 640))
    assert o.linear(rnd(0, 640, dtype=torch.bfloat16), w).shape == (0, 30)
    assert o.gated_linear(rnd(0, 640), w).shape == (0, 15)
    for x in (rnd(2, 639), rnd(2, 640, dtype=torch.float16), rnd(2, 1280)[:, ::2], rnd(640)):
        with pytest.raises(OpsError):
            o.linear(x, w)
    with pytest.raises(OpsError):
        o.gated_linear(rnd(2, 640), Int8Weight.quantize(rnd(31, 640)))
    with pytest.raises(OpsError):
        o.gated_linear(rnd(2, 640), w, row_scale=torch.ones(2, device=DEV))
    with pytest.raises(OpsError):
        o.gated_linear(rnd(2, 640), w, "relu2")


@gpu
def test_tensors_on_another_device_than_the_current_one_are_refused(monkeypatch):
    from qwen3_runtime_amd.ops import OpsError, hip

    o, w, x = ops(), Int8Weight.quantize(rnd(32, 640)), rnd(2, 640)
    o.linear(x, w)
    monkeypatch.setattr(hip, "_raw_device", lambda: 1)  # as if another device were current
    for call in (lambda: o.linear(x, w), lambda: o.gated_linear(x, w), lambda: o.quantize_rows(x),
                 lambda: o.add_rmsnorm_codes(x.clone(), None, torch.ones(640, device=DEV), 1e-6, torch.float32)):
        with pytest.raises(OpsError, match="current device"):
            call()


@gpu
@pytest.mark.parametrize("offset", [1, 2, 8])
@pytest.mark.parametrize("m", [1, 5, 70])
def test_rows_that_begin_anywhere(m, offset):
    w = Int8Weight.quantize(rnd(48, 640, seed=2))
    x = rnd(m * 640 + offset, seed=1, dtype=torch.bfloat16)[offset:].view(m, 640)
    near(ops().linear(x, w), product(x, w), torch.bfloat16)
    # and weights: columns of a wider matrix, rows that begin anywhere
    wide = torch.randint(-127, 128, (48, 700), dtype=torch.int8, generator=torch.Generator().manual_seed(3)).to(DEV)
    w = Int8Weight(wide[:, offset: offset + 640], torch.ones(96, device=DEV)[::2])
    near(ops().linear(x, w), product(x, w), torch.bfloat16)


# ---- needs no GPU


def test_a_weight_in_8_bits():
    w = rnd(7, 130, seed=5, device="cpu", dtype=torch.bfloat16)
    w[3] = 0
    q = Int8Weight.quantize(w)
    assert q.shape == (7, 130) and q.width == 256 and q.values.shape == (7, 256) and not q.values[:, 130:].any()
    assert q.num_bytes == 7 * 256 + 28
    off = (q.values[:, :130].float() * q.scale[:, None] - w.float()).abs()
    assert bool((off <= q.scale[:, None] * (0.5 + 1e-4)).all()) and not q.values[3].any()
    # held as it is where it can be
    v = torch.ones(4, 256, dtype=torch.int8)
    assert Int8Weight(v, torch.ones(4)).values is v


@pytest.mark.parametrize("values,scale", [
    (torch.zeros(4, 8), torch.ones(4)), (torch.zeros(4, dtype=torch.int8), torch.ones(4)), (torch.zeros(4, 8, dtype=torch.int8), torch.ones(3)),
    (torch.zeros(4, 8, dtype=torch.int8), torch.ones(4, dtype=torch.float64)), (torch.zeros(0, 8, dtype=torch.int8), torch.ones(0)),
    (torch.zeros(1, (1 << 17) + 1, dtype=torch.int8), torch.ones(1))])
def test_a_weight_in_8_bits_refuses(values, scale):
    with pytest.raises(ValueError):
        Int8Weight(values, scale)


def test_a_weight_that_is_not_finite_is_refused():
    w = torch.ones(3, 4)
    w[1, 2] = float("nan")
    with pytest.raises(ValueError, match="infinity or a NaN"):
        Int8Weight.quantize(w)
    with pytest.raises(ValueError):
        Int8Weight.quantize(torch.ones(3, 4, dtype=torch.int32))


def test_planes_refuse_on_the_host():
    from ctypes import c_void_p

    from qwen3_runtime_amd.ops.hip import HipOps

    lib, p = HipOps().lib, c_void_p(1 << 20)  # not read: the sizes are refused
    planes = lambda m, n, k, width, tile=12, parts=2, x=p, work=p: lib.qrt_int8_planes(x, 1, p, p, p, p, work, m, n, k, width, tile, parts, None)  # noqa: E731
    for bad in (dict(parts=1), dict(parts=0), dict(parts=-2), dict(parts=65), dict(parts=5), dict(parts=3), dict(tile=14), dict(x=c_void_p(8))):
        assert planes(40, 64, 512, 512, **bad) != 0, bad
    for bad in ((40, 0, 512, 512), (40, 64, 512, 500), (-1, 64, 512, 512)):
        assert planes(*bad) != 0, bad


def test_entry_points_refuse_sizes_on_the_host():
    from ctypes import c_int, c_void_p

    from qwen3_runtime_amd.ops.hip import HipOps

    lib, p = HipOps().lib, c_void_p(1 << 20)  # not read: the sizes are refused
    product = lambda m, n, k, width, tile=0, act=-1, dtype=1, out=1, work=p, x=p, codes=None: lib.qrt_int8_product(  # noqa: E731
        x, dtype, codes, p, p, p, out, work, m, n, k, width, tile, act, 0.0, None)
    for bad in ((1, 0, 128, 128), (1, 16, 128, 100), (1, 16, 200, 128), (1, 16, 0, 128), (1, 16, 1 << 18, 1 << 18), (-1, 16, 128, 128)):
        assert product(*bad) != 0, bad
    for bad in (dict(act=2), dict(dtype=2), dict(out=2), dict(work=None), dict(work=c_void_p(8))):
        assert product(5, 16, 128, 128, **bad) != 0, bad
    assert product(1, 16, 128, 128, x=c_void_p((1 << 20) + 2)) != 0 and product(9, 16, 128, 128, x=c_void_p((1 << 20) + 2), codes=p) != 0
    quantize = lambda m, k, width, dtype=1: lib.qrt_quantize_rows(p, c_int(dtype), p, p, c_int(m), c_int(k), c_int(width), None)  # noqa: E731
    for bad in ((1, 129, 128), (1, 0, 128), (-1, 128, 128), (1, 128, 136), (1, 128, 128, 2)):
        assert quantize(*bad) != 0
