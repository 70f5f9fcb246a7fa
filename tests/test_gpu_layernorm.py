"""uemda_amd.norm on the device against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                        # half a step of fp32, relative


def reference(x, w, b, dy, eps):
    """everything in 64 bits: y, dx, dw, db and the quantities the error bounds are made of"""
    x, dy = x.double(), dy.double()
    w64 = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    mu = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    hat = (x - mu) * rstd
    y = hat * w64 + (0 if b is None else b.double())
    g = dy * w64
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return y, dx, (dy * hat).sum(0), dy.sum(0), hat, rstd, g, w64


def bounds(x, dy, b, r):
    """First-order error bounds.  A sum of C terms runs over a lane's elements (at most C / 64 + 32) and a tree of 8 exchanges: D roundings
    of half a step each, relative to the sum of magnitudes.  D + 8 covers the rounding of 1 / C, of the root and of the products."""
    y, dx, dw, db, hat, rstd, g, w = r
    rows, c = x.shape
    D = c / 64 + 32 + 8 + 8
    ax = x.double().abs().mean(1, keepdim=True) * rstd                         # the mean's error reaches hat through rstd
    ehat = U * (D * ax + 2 * D * hat.abs() + D * ax * (hat.abs() + 1) * hat.abs().clamp(max=1))
    ey = ehat * w.abs() + 2 * U * (y.abs() + (0 if b is None else b.double().abs()))
    gm, ghm = g.abs().mean(1, keepdim=True), (g * hat).abs().mean(1, keepdim=True)
    edx = rstd * (U * D * (g.abs() + 2 * gm + 3 * hat.abs() * ghm) + ehat * ghm + hat.abs() * (g.abs() * ehat).mean(1, keepdim=True)) \
        + 2 * D * U * dx.abs()
    Dr = rows / 64 + 64                                                        # a team's rows, then the teams', waves' and blocks' sums
    edw = (dy.double().abs() * ehat).sum(0) + U * Dr * (dy.double() * hat).abs().sum(0)
    edb = U * Dr * dy.double().abs().sum(0)
    return ey, edx, edw, edb


def close(got, want, bound, what):
    assert got.shape == want.shape, what
    step = torch.finfo(got.dtype).eps / 2
    tol = bound * (1 + 2 * step) + step * want.abs() + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol).max()))


def data(rows, c, dtype, seed, offset=0.0, pdtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) * (torch.rand(rows, 1, generator=g) * 2 + 0.1) + torch.randn(rows, 1, generator=g) + offset).to(dtype)
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).to(pdtype), (0.2 * torch.randn(c, generator=g)).to(pdtype)
    dy = torch.randn(rows, c, generator=g).to(dtype)
    return x.cuda(), w.cuda(), b.cuda(), dy.cuda()


def check(x, w, b, dy, eps=1e-5):
    from uemda_amd.norm import layer_norm
    c = x.shape[-1]
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    need = [t for t in leaves if t is not None]
    grads = dict(zip(["x"] + ["w"] * (w is not None) + ["b"] * (b is not None), torch.autograd.grad(y, need, dy)))
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)                        # inference form: the same numbers
    x2, dy2 = x.reshape(-1, c), dy.reshape(-1, c)
    r = reference(x2, w, b, dy2, eps)
    ey, edx, edw, edb = bounds(x2, dy2, b, r)
    close(y.detach().reshape(-1, c), r[0], ey, "y")
    close(grads["x"].reshape(-1, c), r[1], edx, "dx")
    if w is not None:
        close(grads["w"], r[2], edw, "dw")
    if b is not None:
        close(grads["b"], r[3], edb, "db")
    return y, grads


SIZES = [(1, 1), (3, 1), (1, 2), (5, 8), (7, 9), (1000, 7), (33, 64), (17, 100), (130, 128), (129, 256), (64, 257), (66, 260), (300, 777),
         (41, 1001), (1031, 96), (12, 1024), (9, 1026), (33, 2048), (17, 2049), (9, 4100), (7, 5000), (3, 8192), (2, 8191), (2, 8200), (2, 20001),
         (1, 2048), (9000, 48), (5000, 513), (100, 33), (40001, 33), (1000, 50), (3001, 17), (20, 13), (5000, 67), (129, 131), (77, 203), (5001, 255)]


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_and_its_gradients(rows, c, dtype):
    check(*data(rows, c, dtype, rows * 31 + c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("have", ["wb", "w", "b", ""])
def test_optional_and_16_bit_parameters(dtype, have):
    x, w, b, dy = data(50, 200, dtype, 3, pdtype=torch.bfloat16)
    check(x, w if "w" in have else None, b if "b" in have else None, dy)


@pytest.mark.parametrize("c", [2048, 777, 120, 33])
def test_maps_of_more_than_2_to_the_31_elements(c):
    """every row's y and dx, and the parameter gradients over all of them, checked a slice at a time"""
    from uemda_amd.norm import layer_norm
    rows, part = (2 ** 31 + 2 ** 24) // c, 2 ** 27 // c
    gen = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(rows, c, generator=gen, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(rows, c, generator=gen, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(c, generator=gen, device="cuda").requires_grad_()
    b = torch.randn(c, generator=gen, device="cuda").requires_grad_()
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    sums = [torch.zeros(c, dtype=torch.float64, device="cuda") for _ in range(4)]
    Dr = rows / 64 + 64
    with torch.no_grad():
        for at in list(range(0, rows, part)):
            s = slice(at, min(rows, at + part))
            r = reference(x[s], w, b, dy[s], 1e-5)
            ey, edx, edw, edb = bounds(x[s], dy[s], b, r)
            close(y[s], r[0], ey, "y")
            close(dx[s], r[1], edx, "dx")
            mag = dy[s].double().abs().sum(0), (dy[s].double() * r[4]).abs().sum(0)
            for t, v in zip(sums, (r[2], edw + U * Dr * mag[1], r[3], edb + U * Dr * mag[0])):
                t += v
            del r, ey, edx
    close(dw, sums[0], sums[1], "dw")
    close(db, sums[2], sums[3], "db")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_mean_far_from_zero_keeps_its_variance(dtype):
    check(*data(40, 640, dtype, 5, offset=100.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,start", [(8, 0), (3, 0), (0, 1), (5, 2)])
@pytest.mark.parametrize("c", [64, 512, 777, 2048])
def test_strided_rows_and_unaligned_starts(dtype, pad, start, c):
    """x and dy as column slices of wider buffers, beginning anywhere; what lies between the rows is not touched or read into the result"""
    rows = 21
    x, w, b, dy = data(rows, c, dtype, c + pad)
    wide = torch.full((rows, c + pad + start), float("nan"), device="cuda", dtype=dtype)
    wide[:, start:start + c] = x
    wdy = torch.full_like(wide, float("nan"))
    wdy[:, start:start + c] = dy
    y, g = check(wide[:, start:start + c], w, b, wdy[:, start:start + c])
    y0, g0 = check(x, w, b, dy)
    shift = torch.empty(rows * c + start, device="cuda", dtype=dtype)[start:].view(rows, c).copy_(x)      # dense, but off the 16-byte grid
    check(shift, w, b, dy)
    # neither changes the values beyond the order of the sums
    tol = 1e-5 if dtype == torch.float32 else 2.0 ** -7
    torch.testing.assert_close(y, y0, rtol=tol, atol=tol)


def test_leading_dimensions_empty_batches_and_broadcast_gradients():
    from uemda_amd.norm import LayerNorm, layer_norm
    x, w, b, dy = data(24, 72, torch.float32, 9)
    check(x.view(2, 3, 4, 72), w, b, dy.view(2, 3, 4, 72))
    check(x.view(2, 12, 72).transpose(0, 1), w, b, dy.view(12, 2, 72))
    xl, wl, bl = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    layer_norm(xl, wl, bl).sum().backward()                                    # dy is a broadcast scalar
    r = reference(x, w, b, torch.ones_like(x), 1e-5)
    _, edx, edw, _ = bounds(x, torch.ones_like(x), b, r)
    close(xl.grad, r[1], edx, "dx")
    close(wl.grad, r[2], edw, "dw")
    assert torch.equal(bl.grad, torch.full_like(b, 24.0))
    e = torch.empty(0, 72, device="cuda", requires_grad=True)
    out = layer_norm(e, wl, bl)
    gw, = torch.autograd.grad(out, [wl], torch.empty_like(out))
    assert out.shape == (0, 72) and not gw.any()
    m = LayerNorm(72, channel_dim=1).cuda()
    fm = x.view(2, 3, 4, 72).permute(0, 3, 1, 2)                               # a logical NCHW map in channels_last memory
    out = m(fm)
    assert out.shape == fm.shape and out.is_contiguous(memory_format=torch.channels_last)
    close(out.detach().permute(0, 2, 3, 1).reshape(24, 72), reference(x, None, None, dy, 1e-5)[0], bounds(x, dy, None, reference(x, None, None, dy, 1e-5))[0], "map")
    assert torch.equal(m(fm.contiguous()), out)
    assert list(LayerNorm(5).state_dict()) == ["weight", "bias"] and not list(LayerNorm(5, affine=False).parameters())


def test_non_finite_rows_stay_in_their_rows():
    from uemda_amd.norm import layer_norm
    x, w, b, dy = data(10, 300, torch.float32, 11)
    clean = layer_norm(x, w, b)
    x[3, 7], x[8, 299] = float("nan"), float("inf")
    got = layer_norm(x, w, b)
    keep = torch.ones(10, dtype=torch.bool)
    keep[3] = keep[8] = False
    assert torch.equal(got[keep], clean[keep]) and got[3].isnan().all() and got[8].isnan().all()
    same = torch.full((4, 96), 3.0, device="cuda")                             # a row without variance: exactly its bias
    assert torch.equal(layer_norm(same, w[:96], b[:96]), b[:96].expand(4, 96))


def test_gradient_against_differences():
    """the kernel's gradient along a direction against the kernel's own forward, moved both ways"""
    from uemda_amd.norm import layer_norm
    x, w, b, dy = data(6, 40, torch.float32, 13)
    _, g = check(x, w, b, dy)
    h = 2.0 ** -7
    r = reference(x, w, b, dy, 1e-5)
    ey = bounds(x, dy, b, r)[0]
    gen = torch.Generator().manual_seed(1)
    for name, t in (("x", x), ("w", w), ("b", b)):
        v = torch.randn(t.shape, generator=gen).sign().cuda()
        args = dict(x=x, w=w, b=b)

        def f(s, double=False):
            a = {k: (u.double() if double else u) for k, u in args.items()}
            a[name] = a[name] + s * h * v
            y = reference(a["x"], a["w"], a["b"], dy, 1e-5)[0] if double else layer_norm(a["x"], a["w"], a["b"]).double()
            return (y * dy.double()).sum()
        got = (f(1) - f(-1)) / (2 * h)
        exact = (g[name].double() * v.double()).sum()
        # the forward's rounding over 2 h (the moved point itself rounds too: one step of x, w or b), and the 64-bit formula's own
        # distance between difference and derivative at this h
        moved = U * (t.abs().max() + h) * 2 * g[name].double().abs().sum() / (2 * h)
        rounding = 2 * (ey * 1.5 * dy.double().abs()).sum() / (2 * h) + moved
        curve = ((f(1, True) - f(-1, True)) / (2 * h) - (dict(x=r[1], w=r[2], b=r[3])[name] * v.double()).sum()).abs()
        assert abs(got - exact) <= rounding + 1.5 * curve + 1e-6, (name, float(got), float(exact), float(rounding), float(curve))


def test_a_second_derivative_is_refused():
    from uemda_amd import UemError
    from uemda_amd.norm import layer_norm
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = layer_norm(x)
    with pytest.raises(UemError, match="gradient of the gradient"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """(the engine would end the process) -- and is fine once that graph is gone"""
    from uemda_amd import UemError
    from uemda_amd.grouped import grouped_linear
    from uemda_amd.norm import layer_norm
    x = torch.randn(6, 16, device="cuda", requires_grad=True)
    w = torch.randn(2, 8, 16, device="cuda", requires_grad=True)
    off = torch.tensor([0, 2, 6], device="cuda")
    dy, dz = torch.randn(6, 16, device="cuda"), torch.randn(6, 8, device="cuda")
    want = torch.autograd.grad(layer_norm(x), x, dy)[0], torch.autograd.grad(grouped_linear(x, w, off), (x, w), dz)
    held = layer_norm(x), grouped_linear(x, w, off)
    for f in (lambda: layer_norm(x), lambda: grouped_linear(x.detach(), w, off)):
        with pytest.raises(UemError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                f()
        torch.cuda.synchronize()
    with torch.no_grad():                                                      # without gradients nothing stands in the way
        free = torch.cuda.CUDAGraph()
        with torch.cuda.graph(free):
            y = layer_norm(x)
        free.replay()
        assert torch.equal(y, held[0])
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer_norm(x), x, dy)[0], torch.autograd.grad(grouped_linear(x, w, off), (x, w), dz)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_streams_of_the_callers_choice():
    """two calls at once on two streams, forward and backward on the stream that is current"""
    from uemda_amd.norm import layer_norm
    sets = [data(2000, 384, torch.float32, 50 + k) for k in range(2)]
    want = []
    for x, w, b, dy in sets:
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = layer_norm(*leaves)
        want.append([y.detach()] + list(torch.autograd.grad(y, leaves, dy)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, (x, w, b, dy) in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                leaves = [t.clone().requires_grad_() for t in (x, w, b)]
                y = layer_norm(*leaves)
                got.append([y.detach()] + list(torch.autograd.grad(y, leaves, dy)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for g, v in zip(got, want) for a, c in zip(g, v))


def test_results_repeat_and_a_captured_step_replays():
    from uemda_amd.norm import layer_norm
    x, w, b, dy = data(4097, 320, torch.bfloat16, 17)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    first = [t.clone() for t in step()]
    assert all(torch.equal(a, c) for a, c in zip(step(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(data(4097, 320, torch.bfloat16, 18 + k)[0])
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, want)), k


def test_a_gradient_with_a_tangent_is_refused():
    """forward mode over a backward pass: the node's kernels would drop the tangent of dy"""
    import torch.autograd.forward_ad as fa

    from uemda_amd import UemError
    from uemda_amd.grouped import grouped_linear
    from uemda_amd.norm import layer_norm
    x = torch.randn(6, 8, device="cuda", requires_grad=True)
    w, off = torch.randn(2, 4, 8, device="cuda"), torch.tensor([0, 3, 6], device="cuda")
    for y in (layer_norm(x), grouped_linear(x, w, off)):
        with fa.dual_level():
            with pytest.raises(UemError, match="forward-mode"):
                torch.autograd.grad(y, x, fa.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
        assert torch.autograd.grad(y, x, torch.ones_like(y))[0].isfinite().all()


def close_bounds(x, dy, b, r, D, Dr):
    """`bounds` where the sums over a row, or over the rows of a column, are kept in 64 bits: D and Dr roundings of half a step, whatever the length"""
    y, dx, dw, db, hat, rstd, g, w = r
    ax = x.double().abs().mean(1, keepdim=True) * rstd
    ehat = U * (D * ax + 2 * D * hat.abs() + D * ax * (hat.abs() + 1) * hat.abs().clamp(max=1))
    ey = ehat * w.abs() + 2 * U * (y.abs() + (0 if b is None else b.double().abs()))
    gm, ghm = g.abs().mean(1, keepdim=True), (g * hat).abs().mean(1, keepdim=True)
    edx = rstd * (U * D * (g.abs() + 2 * gm + 3 * hat.abs() * ghm) + ehat * ghm + hat.abs() * (g.abs() * ehat).mean(1, keepdim=True)) + 2 * D * U * dx.abs()
    edw = (dy.double().abs() * ehat).sum(0) + U * Dr * (dy.double() * hat).abs().sum(0)
    return ey, edx, edw, U * Dr * dy.double().abs().sum(0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [8193, 20001, 1000003, 2 ** 24])
def test_long_rows_keep_their_mean_and_variance(c, dtype):
    """rows beyond the register kernels, of one value, of values far from zero, of a deviation under the mean's 32-bit sum's error.  Roundings on
    the way to hat: the mean, the difference, the variance and its sum with eps, the root, the quotient, the product -- 8 with one to spare"""
    g = torch.Generator(device="cuda").manual_seed(c)
    rows = torch.tensor([[1.1, 0.0], [100.1, 0.01 if dtype == torch.float32 else 1.0], [-7.3, 0.1]], device="cuda")
    x = (rows[:, :1] + rows[:, 1:] * torch.randn(3, c, generator=g, device="cuda")).to(dtype)
    w, b = 1 + 0.2 * torch.randn(c, generator=g, device="cuda"), 0.2 * torch.randn(c, generator=g, device="cuda")
    dy = (1.1 + 0.1 * torch.randn(3, c, generator=g, device="cuda")).to(dtype)
    from uemda_amd.norm import layer_norm
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        r = reference(x, w, b, dy, 1e-5)
        e = close_bounds(x, dy, b, r, 8, 8)
        for got, want, bound, what in zip((y.detach(), *grads), r, e, ("y", "dx", "dw", "db")):
            close(got, want, bound, what)


def test_parameter_gradients_of_many_rows_that_begin_anywhere():
    """sums over 260001 rows of one sign by the pass over columns: 64 bits, its blocks' sums rounded once and added in a tree of less than 32"""
    from uemda_amd.norm import layer_norm
    rows, c = 260001, 300
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, c + 1, generator=g, device="cuda")[:, 1:]
    dy = torch.full((rows, c + 1), 1.1, device="cuda")[:, 1:]
    w, b = torch.ones(c, device="cuda", requires_grad=True), torch.zeros(c, device="cuda", requires_grad=True)
    grads = torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)
    with torch.no_grad():
        r = reference(x, w, b, dy, 1e-5)
        e = close_bounds(x, dy, b, r, c / 64 + 48, 32)
        close(grads[0], r[2], e[2], "dw")
        close(grads[1], r[3], e[3], "db")


def test_rows_of_more_columns_than_a_launch_has_threads_for():
    """the parameter gradients of 2^25 + 3 columns: 16 columns to a block of 1024 threads would be more than 2^32 threads"""
    from uemda_amd.norm import layer_norm
    c = 2 ** 25 + 3
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(2, c, generator=g, device="cuda") for _ in range(2))
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        r = reference(x, w, b, dy, 1e-5)
        for got, want, bound, what in zip((y.detach(), *grads), r, close_bounds(x, dy, b, r, 8, 8), ("y", "dx", "dw", "db")):
            close(got, want, bound, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_map_without_one_row_stride_is_copied_once(dtype):
    """contiguous NCHW through channel_dim = 1: the forward's copy is what the backward pass reads, so that it takes memory for dx alone (and the
    parameter gradients' sums, less than a quarter of a map here); and the gradient is that of the values that went in"""
    from uemda_amd.norm import LayerNorm
    g = torch.Generator().manual_seed(2)
    ln = LayerNorm(64, channel_dim=1).cuda()
    x = torch.randn(4, 64, 96, 100, generator=g).to(dtype).cuda()
    dy = torch.randn(4, 64, 96, 100, generator=g).to(dtype).cuda().contiguous(memory_format=torch.channels_last)
    ref = [t.clone() for t in torch.autograd.grad(ln(x.clone().contiguous(memory_format=torch.channels_last).requires_grad_()), list(ln.parameters()), dy)]
    leaf = x.clone().requires_grad_()
    into = leaf * 1
    y = ln(into)
    with torch.no_grad():
        into.mul_(float("nan"))                                                # (the node holds the copy: this is allowed, and changes nothing)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    dx, *grads = torch.autograd.grad(y, [into, *ln.parameters()], dy)
    peak = torch.cuda.max_memory_allocated() - before
    assert peak < 1.25 * x.numel() * x.element_size(), peak / (x.numel() * x.element_size())
    assert all(torch.equal(p, q) for p, q in zip(grads, ref)) and dx.isfinite().all()
