"""Group normalisation with an activation on the GPU, forward and backward, against the formula in float64.

Tolerances, e = 2^-24 (half a step of f32, relative). Forward: z is one f64 FMA, rounded once (e |z|, which moves an
activation by at most (1 + |z|) e relative). swish: exp's argument -z log2(e) carries 2 e |z|, exp2 and 1/x one unit in
the last place (2 e) each, 1 + exp and the product e each: (7 + 3 |z|) e in all, taken as 8 (1 + |z|) e. bf16 outputs
add half a step, 2^-8 relative. Statistics: f64 sums, rounded once.
Backward: the slope of swish, s (1 + z (1 - s)), carries at most 16 (1 + |z|)^2 e s by the same count. A thread sums up
to 64 values in f32 (64 e of the sum of their sizes), partials are rounded once more: 70 e of the sum of sizes covers a
sum. h carries 2 e, dx = rstd (scale dz - c1 - h c2) four roundings of its terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
ACTS = ["linear", "relu", "swish", "hard_swish"]
# (B, H, W, C, groups)
SHAPES = [(1, 1, 1, 1, 1),             # one value: variance 0
          (2, 1, 1, 8, 2),             # one pixel
          (1, 15, 30, 96, 8),          # groups of 12: no whole 16-byte vectors of bf16
          (2, 9, 7, 24, 24),           # instance norm
          (3, 61, 53, 42, 7),          # 6-channel groups
          (2, 5, 3, 3, 1), (1, 40, 30, 5, 5), (2, 33, 17, 7, 1),      # channel counts that no vector divides
          (2, 120, 120, 128, 32),      # several tiles
          (1, 6, 5, 2200, 4),          # several channel blocks, groups across their borders
          (1, 3, 3, 1030, 2), (1, 4, 4, 2048, 1), (1, 2, 3, 1500, 1500),
          (300, 2, 2, 16, 4),          # many small images
          (1, 300, 301, 2, 1),         # few channels, many pixels
          (300, 50, 42, 4, 2),         # more images than workgroups, two passes each
          (1, 42, 50, 1025, 5),        # two passes over two channel blocks, a group across their border
          (1, 42, 50, 1500, 1500),     # more groups than the second pass merges by itself
          (1, 50, 60, 4400, 11),       # whole vectors in two channel blocks
          (2, 480, 480, 80, 5)]        # past the caches


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("needs a GPU")


def _op():
    from realtime_style_transfer_amd.styleTransfer import group_norm, group_norm_gradients
    return group_norm, group_norm_gradients


def _inputs(shape, dtype, per_image, seed=0, mean=1.0):
    B, H, W, C, G = shape
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, H, W, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + mean * torch.randn(C, generator=g))
    aff = (B, C) if per_image else (C,)
    scale, bias = 1 + 0.3 * torch.randn(*aff, generator=g), 0.5 * torch.randn(*aff, generator=g)
    dy = torch.randn(B, H, W, C, generator=g)
    return x.to(dtype).cuda(), scale.cuda(), bias.cuda(), dy.to(dtype).cuda()


def _wide(t, B, C):       # (C,) or (B, C) -> (B, 1, C)
    return t.double().expand(B, C)[:, None]


def _stats64(x, G, eps):
    B, H, W, C = x.shape
    r = x.double().reshape(B, H * W, G, C // G)
    mean = r.mean((1, 3))
    var = ((r - mean[:, None, :, None]) ** 2).mean((1, 3))
    return mean, 1 / torch.sqrt(var + eps)


def _act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "swish":
        return z / (1 + torch.exp(-z))
    if act == "hard_swish":
        return torch.where(z >= 3, z, torch.where(z <= -3, torch.zeros_like(z), z * (z + 3) / 6))
    return z


def _slope64(z, act):
    """The slope and the error its f32 form may have."""
    if act == "relu":
        return (z > 0).double(), torch.zeros_like(z)
    if act == "swish":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s)), 16 * (1 + z.abs()) ** 2 * E * s
    if act == "hard_swish":
        return torch.where(z >= 3, 1.0, torch.where(z > -3, z / 3 + 0.5, 0.0)), 4 * E * (1 + z.abs())
    return torch.ones_like(z), torch.zeros_like(z)


def _forward64(x, scale, bias, G, act, eps=1e-5):
    B, H, W, C = x.shape
    mean, rstd = _stats64(x, G, eps)
    spread = lambda t: t.repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    z = (x.double().reshape(B, H * W, C) - spread(mean)) * spread(rstd) * _wide(scale, B, C) + _wide(bias, B, C)
    return _act64(z, act).view(x.shape), z.view(x.shape), mean, rstd


def _backward64(x, dy, scale, bias, mean, rstd, G, act):
    """-> [(value, tolerance)] of dx, dscale, dbias"""
    B, H, W, C = x.shape
    cg, n = C // G, H * W * (C // G)
    spread = lambda t: t.double().repeat_interleave(cg, 1)[:, None]  # noqa: E731
    group = lambda t: t.sum(1).view(B, G, cg).sum(2).repeat_interleave(cg, 1)[:, None] / n  # noqa: E731
    sc, r = _wide(scale, B, C), spread(rstd)
    h = (x.double().reshape(B, H * W, C) - spread(mean)) * r
    z = h * sc + _wide(bias, B, C)
    slope, se = _slope64(z, act)
    d = dy.double().reshape(B, H * W, C)
    dz, dze = d * slope, d.abs() * (se + 2 * E * slope.abs())
    c1, c2 = group(sc * dz), group(sc * dz * h)
    dx = r * (sc * dz - c1 - h * c2)
    e1 = group(sc.abs() * (dze + 70 * E * dz.abs()))
    e2 = group(sc.abs() * h.abs() * (dze + 74 * E * dz.abs()))
    tol = r * (sc.abs() * dze + e1 + h.abs() * e2 + 4 * E * ((sc * dz).abs() + c1.abs() + (h * c2).abs()))
    keep = (lambda t: t.sum(1)) if scale.dim() == 2 else (lambda t: t.sum((0, 1)))
    half = 2.0 ** -8 if x.dtype is torch.bfloat16 else E
    return [(dx.view(x.shape), (tol + half * dx.abs()).view(x.shape)),
            (keep(dz * h), keep(h.abs() * (dze + 74 * E * dz.abs())) + E * keep(dz * h).abs()),
            (keep(dz), keep(dze + 70 * E * dz.abs()) + E * keep(dz).abs())]


def _near(got, want, tol, what):
    off = (got.double() - want).abs() - tol
    assert bool((off <= 1e-30).all()), f"{what}: {float(off.max()):.3e} beyond its tolerance"


def _check_forward(x, scale, bias, G, act):
    y, mean, rstd = _op()[0](x, scale, bias, G, activation=act, return_statistics=True)
    ref, z, m, r = _forward64(x, scale, bias, G, act)
    half = 2.0 ** -8 if x.dtype is torch.bfloat16 else 0.0
    assert y.dtype is x.dtype and y.shape == x.shape and mean.shape == rstd.shape == (x.shape[0], G)
    # z's own 64 bits, which count where z is next to 0: a sum of n values is off by at most n 2^-53 of the sum of their
    # sizes on either side, so the mean by n 2^-53 max|x|, rstd by twice that relative to itself over var's own scale
    # (max|x| / std >= |x - mean| / std), and z = scale (x - mean) rstd + bias by 4 n 2^-53 (|scale| rstd max|x| + |bias|)
    # times max|x| rstd; slopes are at most 1.1
    n, top = x.numel() // (x.shape[0] * G), float(x.abs().max()) * float(r.max())
    tiny = 5 * n * 2.0 ** -53 * (1 + top) * (float(scale.abs().max()) * top + float(bias.abs().max()))
    _near(y, ref, 8 * (1 + z.abs()) * E * ref.abs() + 2 * E * z.abs() * (act == "hard_swish") + half * ref.abs() + tiny, "y")
    _near(mean, m, E * m.abs() + 1e-12, "mean")
    _near(rstd, r, 2 * E * r, "rstd")
    return y, mean, rstd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    for k, act in enumerate(ACTS):
        x, scale, bias, _ = _inputs(shape, dtype, per_image=k % 2 == 1, seed=k)
        _check_forward(x, scale, bias, shape[-1], act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, dtype):
    for k, act in enumerate(ACTS):
        x, scale, bias, dy = _inputs(shape, dtype, per_image=k % 2 == 0, seed=10 + k)
        G = shape[-1]
        mean, rstd = (t.float() for t in _stats64(x, G, 1e-5))
        got = _op()[1](x, dy, scale, bias, mean, rstd, G, activation=act)
        for what, g, (want, tol) in zip(("dx", "dscale", "dbias"), got, _backward64(x, dy, scale, bias, mean, rstd, G, act)):
            assert g.shape == want.shape
            _near(g, want, tol, what)
        assert got[0].dtype is dtype and got[1].dtype is got[2].dtype is torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_tensors_at_any_alignment(dtype, offset):
    """Views that start inside a buffer: narrower loads, the same values."""
    shape = (2, 11, 9, 32, 8)
    x, scale, bias, dy = _inputs(shape, dtype, False)
    shift = lambda t: torch.cat([t.new_zeros(offset), t.reshape(-1)])[offset:].view(t.shape)  # noqa: E731
    _check_forward(shift(x), scale, bias, 8, "swish")
    mean, rstd = (t.float() for t in _stats64(x, 8, 1e-5))
    for g, (want, tol) in zip(_op()[1](shift(x), shift(dy), shift(scale), shift(bias), shift(mean), rstd, 8, "swish"),
                              _backward64(x, dy, scale, bias, mean, rstd, 8, "swish")):
        _near(g, want, tol, "gradient")


def test_other_memory_orders():
    """A channels-first tensor is read as the channels-last one it stands for; a strided dy too."""
    x, scale, bias, dy = _inputs((2, 8, 6, 16, 4), torch.float32, True)
    first = x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert not first.is_contiguous()
    gn, grad = _op()
    y, mean, rstd = gn(x, scale, bias, 4, activation="relu", return_statistics=True)
    assert torch.equal(gn(first, scale, bias, 4, activation="relu"), y)
    a = grad(x, dy, scale, bias, mean, rstd, 4, "relu")
    b = grad(first, dy.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), scale, bias, mean, rstd, 4, "relu")
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_large_mean_keeps_the_variance():
    """mean / std = 10^4: E[x^2] - mean^2 in 32 bits would have no digit left."""
    x, scale, bias, _ = _inputs((2, 30, 40, 32, 4), torch.float32, False)
    x = (x + 1e4).contiguous()
    y, mean, rstd = _op()[0](x, scale, bias, 4, return_statistics=True)
    ref, z, m, r = _forward64(x, scale, bias, 4, "linear")
    _near(rstd, r, 2 * E * r, "rstd")
    _near(y, ref, 2 * E * ref.abs() + 1e-7, "y")     # z = a x + c in f64: c ~ 10^4 a rounds to 10^4 2^-53


@pytest.mark.parametrize("bad", [float('nan'), float('inf')])
def test_a_bad_value_stays_in_its_group(bad):
    x, scale, bias, dy = _inputs((3, 7, 5, 16, 4), torch.float32, False)
    clean = _op()[0](x, scale, bias, 4, activation="relu")
    x[1, 3, 2, 6] = bad                                # image 1, group 1
    y, mean, rstd = _op()[0](x, scale, bias, 4, activation="relu", return_statistics=True)
    keep = torch.ones(3, 16, dtype=torch.bool, device='cuda')
    keep[1, 4:8] = False
    keep = keep[:, None, None].expand_as(y)
    assert torch.equal(y[keep], clean[keep])
    assert bool(torch.isnan(mean[1, 1]) | torch.isinf(mean[1, 1])) and bool(torch.isnan(y[1, 3, 2, 6]))
    assert int((~torch.isfinite(mean)).sum()) == 1


def test_empty_tensors():
    gn, grad = _op()
    s = torch.ones(8, device='cuda')
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        x = torch.zeros(shape, device='cuda')
        y, mean, rstd = gn(x, s, s, 2, return_statistics=True)
        assert y.shape == shape
        st = torch.zeros(shape[0], 2, device='cuda')
        dx, ds, db = grad(x, x, s, s, st, st, 2)
        assert dx.shape == shape and not ds.any() and not db.any()


def test_same_bits_every_time_in_graphs_and_on_other_streams():
    gn, grad = _op()
    x, scale, bias, dy = _inputs((2, 60, 50, 64, 16), torch.bfloat16, True)
    y, mean, rstd = gn(x, scale, bias, 16, activation="swish", return_statistics=True)
    want = (y, *grad(x, dy, scale, bias, mean, rstd, 16, "swish"))

    def run():
        y, m, r = gn(x, scale, bias, 16, activation="swish", return_statistics=True)
        return (y, *grad(x, dy, scale, bias, m, r, 16, "swish"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    both = run()                                       # two calls at once
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, other, both))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, held, eager))


@pytest.mark.parametrize("H", [40, 90])              # one launch, two passes
def test_in_place_through_the_c_interface(H):
    """y may be x, dx may be dy."""
    from realtime_style_transfer_amd import _lib as L
    gn, grad = _op()
    lib = L.load()
    x, scale, bias, dy = _inputs((2, H, 50, 24, 3), torch.float32, False)
    n = H * 50
    y, mean, rstd = gn(x, scale, bias, 3, activation="relu", return_statistics=True)
    dx, ds, db = grad(x, dy, scale, bias, mean, rstd, 3, "relu")
    need = max(lib.rst_group_norm_workspace_size(2, n, 24, 3), lib.rst_group_norm_backward_workspace_size(2, n, 24, 3))
    ws = torch.empty(need, dtype=torch.uint8, device='cuda')
    d2, s2, b2 = dy.clone(), torch.empty_like(ds), torch.empty_like(db)
    L.check(lib.rst_group_norm_backward(x.data_ptr(), d2.data_ptr(), 0, 2, n, 24, 3, scale.data_ptr(),
                                        bias.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), 1, d2.data_ptr(),
                                        s2.data_ptr(), b2.data_ptr(), ws.data_ptr(), L.stream_ptr()))
    x2 = x.clone()
    L.check(lib.rst_group_norm(x2.data_ptr(), 0, 2, n, 24, 3, scale.data_ptr(), bias.data_ptr(), 0, 1e-5, 1,
                               x2.data_ptr(), None, None, ws.data_ptr(), L.stream_ptr()))
    torch.cuda.synchronize()
    assert torch.equal(x2, y) and torch.equal(d2, dx) and torch.equal(s2, ds) and torch.equal(b2, db)


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """The directional derivative of sum(w y) from two forward passes h apart. Its error: the third derivative's h^2 and
    the outputs' rounding, sqrt(N) e |w y| / h ~ 60 * 6e-8 / 2e-2 ~ 2e-4 of |w y|; 5e-3 of the derivative's size covers
    both. An element whose z crosses a kink between the two passes adds at most w, times the jump of the slope there (1
    for relu, 1/2 for hard_swish), times its share of the path: |z(h) - z(-h)| / 2h."""
    gn, grad = _op()
    x, scale, bias, w = _inputs((2, 8, 7, 32, 4), torch.float32, True, seed=3)
    g = torch.Generator().manual_seed(8)
    vx, vs, vb = (torch.randn(t.shape, generator=g).cuda() for t in (x, scale, bias))
    y, mean, rstd = gn(x, scale, bias, 4, activation=act, return_statistics=True)
    dx, ds, db = grad(x, w, scale, bias, mean, rstd, 4, act)
    h = 2e-3
    loss = lambda s: float((w.double() * gn(x + s * vx, scale + s * vs, bias + s * vb, 4, activation=act).double()).sum())  # noqa: E731
    parts = [(dx.double() * vx).sum(), (ds.double() * vs).sum(), (db.double() * vb).sum()]
    want = (loss(h) - loss(-h)) / (2 * h)
    size = float((dx.double() * vx).norm() + (ds.double() * vs).norm() + (db.double() * vb).norm())
    z = [_forward64(x + s * vx, scale + s * vs, bias + s * vb, 4, act)[1] for s in (h, -h)]
    kinks = {"relu": [(0.0, 1.0)], "hard_swish": [(-3.0, 0.5), (3.0, 0.5)]}.get(act, [])
    kink = sum(float((w.double() * (z[0] - z[1]))[(z[0] > at) != (z[1] > at)].abs().sum()) * jump / (2 * h)
               for at, jump in kinks)
    assert abs(float(sum(parts)) - want) < 5e-3 * size + kink, (float(sum(parts)), want, size, kink)


def test_equals_instance_norm_at_one_channel_per_group():
    from realtime_style_transfer_amd.styleTransfer import instance_norm
    x, scale, bias, _ = _inputs((2, 37, 53, 24, 24), torch.float32, True)
    a = instance_norm(x, scale, bias, relu=True)
    b = _op()[0](x, scale, bias, 24, activation="relu")
    ref, z, _, _ = _forward64(x, scale, bias, 24, "relu")
    assert float((b.double() - ref).abs().max()) <= float((a.double() - ref).abs().max()) + 1e-6
    assert float((a - b).abs().max()) < 1e-4           # instance_norm's own bound


def test_offsets_past_32_bits():
    """4.4 G values in one image: elements and bytes beyond 2^32. The statistics by chunks in float64; y, dx at both ends
    and around the 2^32 border from the returned statistics; the affine's gradients by chunks."""
    gn, grad = _op()
    H, W, C, G = 40000, 27500, 4, 2
    x = torch.empty(1, H, W, C, dtype=torch.bfloat16, device='cuda')
    for k in range(0, H, 1000):                        # a different spread and mean along the image
        g = torch.Generator(device='cuda').manual_seed(k)
        x[0, k:k + 1000] = (torch.randn(1000, W, C, generator=g, device='cuda') * (1 + k / H) + k / H).bfloat16()
    scale, bias = torch.tensor([1.0, 0.5, -1.0, 2.0], device='cuda'), torch.tensor([0.1, 0.0, 0.3, -0.2], device='cuda')
    y, mean, rstd = gn(x, scale, bias, G, activation="relu", return_statistics=True)
    s = torch.zeros(2, G, dtype=torch.float64, device='cuda')
    for k in range(0, H, 1000):
        r = x[0, k:k + 1000].double().view(-1, G, 2)
        s += torch.stack([r.sum((0, 2)), (r * r).sum((0, 2))])
    m = s[0] / (H * W * 2)
    _near(mean[0], m, 2 * E * m.abs(), "mean")
    r = 1 / torch.sqrt(s[1] / (H * W * 2) - m * m + 1e-5)
    _near(rstd[0], r, 2 * E * r, "rstd")
    sums = torch.zeros(2, C, dtype=torch.float64, device='cuda')
    size = torch.zeros(2, C, dtype=torch.float64, device='cuda')
    wide = lambda t: t[0].double().repeat_interleave(2)  # noqa: E731

    def chunk(rows):
        xs = x[0, rows].double()
        h = (xs - wide(mean)) * wide(rstd)
        dz = (h * scale.double() + bias.double() > 0) * xs      # dy = x below
        return h, dz
    for k in range(0, H, 1000):
        h, dz = chunk(slice(k, k + 1000))
        sums += torch.stack([(dz * h).sum((0, 1)), dz.sum((0, 1))])
        size += torch.stack([(dz * h).abs().sum((0, 1)), dz.abs().sum((0, 1))])
    dx, dscale, dbias = grad(x, x, scale, bias, mean, rstd, G, "relu")
    _near(dscale, sums[0], 76 * E * size[0], "dscale")
    _near(dbias, sums[1], 72 * E * size[1], "dbias")
    n = H * W * 2
    c1, c2 = ((scale.double() * t).view(G, 2).sum(1).repeat_interleave(2) / n for t in (sums[1], sums[0]))
    a1, a2 = ((scale.double().abs() * t).view(G, 2).sum(1).repeat_interleave(2) / n for t in (size[1], size[0]))
    border = 2 ** 32 // (W * C)
    for rows in (slice(0, 2), slice(border // 2 - 1, border // 2 + 2), slice(border - 1, border + 2), slice(H - 2, H)):
        h, dz = chunk(rows)
        z = h * scale.double() + bias.double()
        _near(y[0, rows], z.clamp(min=0), 2.0 ** -8 * z.abs() + 4 * E * (h.abs() + 1), "y")
        sc, ri = scale.double(), wide(rstd)
        want = ri * (sc * dz - c1 - h * c2)
        _near(dx[0, rows], want, 2.0 ** -8 * want.abs() + ri * 80 * E * ((sc * dz).abs() + a1 + h.abs() * a2), "dx")


def test_refusals_on_the_device():
    gn, grad = _op()
    x, scale, bias, dy = _inputs((2, 4, 4, 8, 2), torch.float32, False)
    st = torch.zeros(2, 2, device='cuda')
    with pytest.raises(ValueError):
        gn(x, scale.cpu(), bias, 2)
    with pytest.raises(ValueError):
        gn(x, scale.bfloat16(), bias, 2)
    with pytest.raises(ValueError):
        gn(x.clone().requires_grad_(), scale, bias, 2)      # autograd would lose it silently
    with torch.no_grad():
        gn(x.clone().requires_grad_(), scale, bias, 2)
    with pytest.raises(ValueError):
        grad(x, dy.bfloat16(), scale, bias, st, st, 2)
    with pytest.raises(ValueError):
        grad(x, dy[:1], scale, bias, st, st, 2)
    with pytest.raises(ValueError):
        grad(x, dy, scale, bias, st[:, :1], st, 2)
    with pytest.raises(ValueError):
        gn(x, scale, bias, 2, eps=-1.0)


def test_an_empty_image_has_no_moments():
    s = torch.ones(8, device='cuda')
    y, mean, rstd = _op()[0](torch.zeros(2, 3, 0, 8, device='cuda'), s, s, 2, return_statistics=True)
    assert y.shape == (2, 3, 0, 8) and bool(mean.isnan().all()) and bool(rstd.isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 37, 53, 24, 6), (3, 5, 5, 32, 32), (8, 4, 4, 64, 8), (9, 4, 4, 64, 8), (4, 16, 16, 256, 32),
                                   (5, 16, 16, 256, 32), (2, 6, 5, 3, 1), (3, 1, 1, 128, 4), (2, 1, 1, 1, 1), (2, 32, 32, 128, 32)])
def test_shared_affine_of_few_small_images(shape, dtype):
    G = shape[-1]
    for k, act in enumerate(ACTS):
        x, scale, bias, dy = _inputs(shape, dtype, per_image=False, seed=40 + k)
        mean, rstd = (t.float() for t in _stats64(x, G, 1e-5))
        got = _op()[1](x, dy, scale, bias, mean, rstd, G, activation=act)
        again = _op()[1](x, dy, scale, bias, mean, rstd, G, activation=act)
        for what, g, h, (want, tol) in zip(("dx", "dscale", "dbias"), got, again,
                                           _backward64(x, dy, scale, bias, mean, rstd, G, act)):
            _near(g, want, tol, what)
            assert torch.equal(g, h)
        for h, g in zip(_backward_in_place(x, dy, scale, bias, mean, rstd, G, k), got):
            assert torch.equal(g, h)


def _backward_in_place(x, dy, scale, bias, mean, rstd, G, act):
    from realtime_style_transfer_amd import _lib as L
    lib, (B, H, W, C) = L.load(), x.shape
    dx, ds, db = dy.clone(), torch.full_like(scale, -1.0), torch.full_like(bias, -1.0)
    ws = torch.empty(lib.rst_group_norm_backward_workspace_size(B, H * W, C, G) + 16, dtype=torch.uint8, device='cuda')
    L.check(lib.rst_group_norm_backward(x.data_ptr(), dx.data_ptr(), int(x.dtype is torch.bfloat16), B, H * W, C, G,
                                        scale.data_ptr(), bias.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), act,
                                        dx.data_ptr(), ds.data_ptr(), db.data_ptr(), ws.data_ptr(), L.stream_ptr()))
    return dx, ds, db


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 4, 9, 8, 4), (1, 90, 45, 8, 4)])       # one launch, two passes
@pytest.mark.parametrize("per_image", [False, True])
def test_the_slope_on_a_kink(shape, dtype, per_image, monkeypatch):
    """z exactly on a kink and one step of x beside it: hard_swish's slope is 1 from z = 3 on and 0 up to z = -3, relu's 0
    at 0. Mean 0 and rstd 1 make z = scale x + bias; with scale 0 every pixel lies on the bias. The side of a kink k is the
    sign of scale x + (bias - k), which 64 bits give exactly: both terms are exact (three-bit scales, small integers) and a
    rounded sum keeps its sign. (z itself would not do: 3 + 1e-30 rounds to 3.)"""
    B, H, W, C, G = shape
    up = 1 + (2.0 ** -7 if dtype is torch.bfloat16 else 2.0 ** -23)
    down = 1 - (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -24)
    points = [s * v for s in (1, -1) for v in (0.0, 3.0, 3 * up, 3 * down, 6.0, 1.5, 3.5, 12.0, 1e-30)]
    x = torch.tensor(points).repeat(-(-B * H * W * C // len(points)))[:B * H * W * C]
    x = x.view(B, C, H, W).permute(0, 2, 3, 1).contiguous().to(dtype).cuda()
    scale = torch.tensor([0.0, 0.0, 1.0, -1.0, 1.0, -1.0, 0.5, -2.0]).cuda()
    bias = torch.tensor([3.0, -3.0, 0.0, 0.0, 3.0, -3.0, 0.0, 3.0]).cuda()
    if per_image:
        scale, bias = (t.expand(B, C).contiguous() for t in (scale, bias))
    dy = _inputs(shape, dtype, False)[3]
    mean, rstd = torch.zeros(B, G, device='cuda'), torch.ones(B, G, device='cuda')

    def slope(z, act):
        from_kink = lambda k: x.double().reshape(B, H * W, C) * _wide(scale, B, C) + (_wide(bias, B, C) - k)  # noqa: E731
        if act == "relu":
            return (from_kink(0.0) > 0).double(), torch.zeros_like(z)
        inside = torch.where(from_kink(-3.0) > 0, z / 3 + 0.5, 0.0)
        return torch.where(from_kink(3.0) >= 0, 1.0, inside), 4 * E * (1 + z.abs())
    monkeypatch.setitem(globals(), "_slope64", slope)
    for act in ("relu", "hard_swish"):
        got = _op()[1](x, dy, scale, bias, mean, rstd, G, activation=act)
        for what, g, (want, tol) in zip(("dx", "dscale", "dbias"), got, _backward64(x, dy, scale, bias, mean, rstd, G, act)):
            _near(g, want, tol, f"{act} {what}")


def test_forward_mode_gradients_are_refused():
    """A tangent would be lost silently, as a recorded gradient would."""
    import torch.autograd.forward_ad as fw
    gn, grad = _op()
    x, scale, bias, dy = _inputs((2, 4, 4, 8, 2), torch.float32, False)
    st = torch.zeros(2, 2, device='cuda')
    with fw.dual_level():
        for k, t in enumerate((x, scale, bias)):
            args = [x, scale, bias]
            args[k] = fw.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match="tangent"):
                gn(*args, 2)
        with pytest.raises(ValueError, match="tangent"):
            grad(x, fw.make_dual(dy, dy), scale, bias, st, st, 2)
        y = gn(x, scale, bias, 2)                       # none of them has one
    assert torch.equal(y, gn(x, scale, bias, 2))


def _device_inputs(shape, per_image, seed):
    B, H, W, C, G = shape
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    aff = (B, C) if per_image else (C,)
    return r(B, H, W, C), 1 + 0.3 * r(*aff), 0.5 * r(*aff), r(B, H, W, C)


# 2^32 threads and more: each kernel's workgroups take several launches
@pytest.mark.parametrize("shape", [(2 ** 22 + 3, 1, 1, 8, 2),          # the two passes of 1024 threads
                                   (61100, 1, 1, 1100, 1100)])         # the merge of 67 M groups, 4 of them in 256 threads
def test_more_workgroups_than_a_launch_takes(shape):
    x, scale, bias, _ = _device_inputs(shape, False, 1)
    _check_forward(x, scale, bias, shape[-1], "swish")


@pytest.mark.parametrize("shape, per_image", [((2 ** 22 + 3, 2, 3, 8, 2), False), ((2 ** 22 + 3, 2, 3, 8, 2), True),
                                              ((2 ** 24 + 5, 1, 1, 4, 1), True)])    # the one-launch form, 256 threads
def test_more_workgroups_than_a_launch_takes_backward(shape, per_image):
    x, scale, bias, dy = _device_inputs(shape, per_image, 2)
    mean, rstd = (t.float() for t in _stats64(x, shape[-1], 1e-5))
    got = _op()[1](x, dy, scale, bias, mean, rstd, shape[-1], activation="relu")
    for what, g, (want, tol) in zip(("dx", "dscale", "dbias"), got,
                                    _backward64(x, dy, scale, bias, mean, rstd, shape[-1], "relu")):
        _near(g, want, tol, what)


@pytest.mark.parametrize("size", [1e25, 1e-25])
@pytest.mark.parametrize("shape", [(2, 7, 9, 24, 3), (1, 90, 45, 8, 4)])       # one launch, two passes
def test_gradients_of_activations_far_from_one(shape, size):
    """rstd^2 and dy (x - mean) are past f32 where dx, dscale and dbias are not."""
    G = shape[-1]
    for act in ACTS:
        x, scale, bias, dy = _inputs(shape, torch.float32, True, seed=50)
        x, dy = x * size, dy * size ** 0.6        # (dx ~ dy / size)
        mean, rstd = (t.float() for t in _stats64(x, G, 0.0))
        got = _op()[1](x, dy, scale, bias, mean, rstd, G, activation=act)
        for what, g, (want, tol) in zip(("dx", "dscale", "dbias"), got, _backward64(x, dy, scale, bias, mean, rstd, G, act)):
            _near(g, want, tol, f"{act} {what}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sums_of_gradients_of_very_different_sizes(dtype):
    """A 32nd of the pixels, those that threads meet first, has gradients of 2^25: added to one of them in 32 bits, the others'
    ones would be lost, 15 e of the sum. The threads' sums are in 64 bits: partials and the result are rounded, 2 e."""
    H, W = 4096, 4096
    x, one = torch.ones(1, H, W, 4, dtype=dtype, device='cuda'), torch.ones(4, device='cuda')
    dy = torch.ones_like(x)
    dy[:, :H // 32] = 2.0 ** 25
    dx, dscale, dbias = _op()[1](x, dy, one, 0 * one, torch.zeros(1, 2, device='cuda'), torch.ones(1, 2, device='cuda'), 2)
    want = dy.double().sum((0, 1, 2))
    for got in (dscale, dbias):
        assert bool(((got.double() - want).abs() <= 2.5 * E * want).all()), float(((got.double() - want) / want).abs().max() / E)
