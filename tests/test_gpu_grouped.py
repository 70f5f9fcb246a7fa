"""uemda_amd.grouped on the device against the groups' products in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def edges(T, lens, head=0):
    """offsets of groups of these lengths behind `head` rows"""
    o = [head]
    for n in lens:
        o.append(o[-1] + n)
    assert o[-1] <= T
    return o


def reference(x, w, b, dy, o):
    """y, dx, dw, db in 64 bits and, beside each, the sums of magnitudes that the accumulators' roundings are relative to"""
    x, w, dy = x.double(), w.double(), dy.double()
    T, K = x.shape
    G, N, _ = w.shape
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=x.device)  # noqa: E731
    y, dx, dw, db, ay, ax, aw, ab = z(T, N), z(T, K), z(G, N, K), z(G, N), z(T, N), z(T, K), z(G, N, K), z(G, N)
    for g in range(G):
        r = slice(o[g], o[g + 1])
        y[r], ay[r] = x[r] @ w[g].t(), x[r].abs() @ w[g].t().abs()
        if b is not None:
            y[r] += b[g].double()
            ay[r] += b[g].double().abs()
        dx[r], ax[r] = dy[r] @ w[g], dy[r].abs() @ w[g].abs()
        dw[g], aw[g] = dy[r].t() @ x[r], dy[r].t().abs() @ x[r].abs()
        db[g], ab[g] = dy[r].sum(0), dy[r].abs().sum(0)
    return (y, ay), (dx, ax), (dw, aw), (db, ab)


def close(got, want, mag, terms, what):
    """a sum of `terms` products kept in fp32: every addition is off by at most one step of the running sum (a matrix instruction may cut
    rather than round), which is at most the sum of magnitudes; then one rounding to the result's type"""
    assert got.shape == want.shape, what
    step = torch.finfo(got.dtype).eps / 2
    tol = 2 * U * (terms + 8) * mag * (1 + step) + step * want.abs() + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol).max()), bad.nonzero()[:4].tolist())


def data(T, G, K, N, dtype, seed, wdtype=None, bdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(dtype)
    w = (torch.randn(G, N, K, generator=g) * K ** -0.5).to(wdtype or dtype)
    b = (0.1 * torch.randn(G, N, generator=g)).to(bdtype or dtype)
    dy = torch.randn(T, N, generator=g).to(dtype)
    return x.cuda(), w.cuda(), b.cuda(), dy.cuda()


def check(x, w, b, dy, o, off_dtype=torch.int32):
    from uemda_amd.grouped import grouped_linear
    T, K = x.shape
    G, N, _ = w.shape
    off = torch.tensor(o, dtype=off_dtype, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    y = grouped_linear(leaves[0], leaves[1], off, leaves[2] if b is not None else None)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(grouped_linear(x, w, off, b), y)
    assert y.dtype == x.dtype and all(g.dtype == t.dtype for g, t in zip(grads, leaves))
    wr = w.to(x.dtype)                                                         # fp32 master weights enter the product rounded
    (ry, ay), (rdx, ax), (rdw, aw), (rdb, ab) = reference(x, wr, b, dy, o)
    lens = torch.tensor([o[g + 1] - o[g] for g in range(G)], dtype=torch.float64, device="cuda")
    close(y.detach(), ry, ay, K + 1, "y")
    close(grads[0], rdx, ax, N, "dx")
    close(grads[1], rdw, aw, lens.view(G, 1, 1), "dw")
    if b is not None:
        close(grads[2], rdb, ab, lens.view(G, 1), "db")
    return y, grads


# T, K, N, lengths of the groups, rows in front
SHAPES = [
    (1, 8, 8, [1], 0),
    (3, 16, 16, [0, 3], 0),
    (5, 64, 32, [0, 0, 0], 2),                       # no group has a row
    (7, 1, 1, [2, 0, 3], 1),
    (9, 2048, 512, [1, 0, 2, 3, 0, 3], 0),           # a few rows: weights are all there is
    (40, 33, 17, [5, 7, 0, 20], 3),                  # odd everything
    (100, 72, 200, [31, 32, 33], 2),
    (257, 64, 129, [128, 129], 0),
    (300, 200, 40, [256, 1, 43], 0),
    (515, 136, 264, [1, 255, 257], 1),
    (700, 77, 333, [100] * 6, 50),
    (1000, 128, 128, [7] * 100, 11),                 # more groups than a wave's lanes
    (640, 24, 136, [1] * 63 + [500] + [2] * 30, 0),
    (2600, 264, 272, [1300, 0, 1290], 5),
    (6000, 320, 320, [5800, 30, 100], 0),            # one group of several chunks in the weight gradient
    (4100, 40, 48, [4100], 0),
    (20000, 24, 16, [19000, 900], 3),                # and of many
    (20001, 23, 17, [20000], 1),
    (50, 40, 1029, [20, 0, 29], 1),                  # few rows and a long reduction, forward and back
    (70, 1031, 600, [33, 1, 0, 32], 0),
    (3, 17, 2050, [1, 2], 0),
    (3500, 40, 136, [3] * 40 + [900] + [0] * 30 + [1100] + [5] * 20 + [256, 512, 300], 4),     # chunks and rests on both sides of lane 64
]


@pytest.mark.parametrize("T,K,N,lens,head", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_and_gradients(T, K, N, lens, head, dtype):
    G = len(lens)
    x, w, b, dy = data(T, G, K, N, dtype, T + K)
    check(x, w, b, dy, edges(T, lens, head))


@pytest.mark.parametrize("T,K,N,lens", [(12800, 512, 520, [5000, 0, 4000, 3000, 800]), (9000, 776, 1000, [3000, 3000, 2999])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_that_take_the_largest_tiles(T, K, N, lens, dtype):
    x, w, b, dy = data(T, len(lens), K, N, dtype, T)
    check(x, w, b, dy, edges(T, lens))


@pytest.mark.parametrize("K,N", [(2048, 24), (40, 2048)])
def test_rows_of_more_than_2_to_the_31_elements(K, N):
    """x and dx, or y and dy, beyond 2^31 elements: the last groups, whose rows lie behind that, and their gradients"""
    from uemda_amd.grouped import grouped_linear
    T = 2 ** 31 // 2048 + 9000
    o = [100, T - 7000, T - 4000, T - 1000]
    gen = torch.Generator(device="cuda").manual_seed(K)
    x, dy = (torch.randn(T, n, generator=gen, device="cuda", dtype=torch.bfloat16) for n in (K, N))
    w, b = torch.randn(3, N, K, generator=gen, device="cuda", dtype=torch.bfloat16), torch.randn(3, N, generator=gen, device="cuda", dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = grouped_linear(x, w, torch.tensor(o, device="cuda"), b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        at = T - 8000                                                          # the end of the first group, the others, and the tail
        (ry, ay), (rdx, ax), (rdw, aw), (rdb, ab) = reference(x[at:], w, b, dy[at:], [0, 1000, 4000, 7000])
        close(y[at:], ry, ay, K + 1, "y")
        close(dx[at:], rdx, ax, N, "dx")
        close(dw[1:], rdw[1:], aw[1:], 3000, "dw")
        close(db[1:], rdb[1:], ab[1:], 3000, "db")
        assert not y[:100].any() and not dx[:100].any()
        want, mag = 0, 0
        for s in range(o[0], o[1], 2 ** 17):                                   # the first group's gradients: nearly all of the rows
            e = min(o[1], s + 2 ** 17)
            want = want + dy[s:e].double().sum(0)
            mag = mag + dy[s:e].double().abs().sum(0)
        close(db[0], want, mag, o[1] - o[0], "db of the long group")


def test_master_weights_int64_offsets_and_no_bias():
    o = edges(200, [60, 0, 100], 7)
    x, w, b, dy = data(200, 3, 48, 56, torch.bfloat16, 1, wdtype=torch.float32, bdtype=torch.float32)
    check(x, w, b, dy, o, torch.int64)
    check(x, w, None, dy, o)
    x, w, b, dy = data(200, 3, 48, 56, torch.float32, 2, bdtype=torch.bfloat16)
    check(x, w, b, dy, o, torch.int64)


def test_master_weights_with_gaps():
    """fp32 weights that are a slice of a wider buffer, under bf16 rows: rounded row by row, what lies between is not read"""
    o = edges(200, [60, 0, 100], 7)
    x, w, b, dy = data(200, 3, 48, 56, torch.bfloat16, 1, wdtype=torch.float32)
    wide = torch.full((3, 56, 53), float("nan"), device="cuda")
    wide[:, :, 2:50] = w
    tall = torch.full((3, 60, 48), float("nan"), device="cuda")
    tall[:, 3:59] = w
    y0, g0 = check(x, w, b, dy, o)
    for v in (wide[:, :, 2:50], tall[:, 3:59], w.transpose(1, 2).contiguous().transpose(1, 2)):
        y, g = check(x, v, b, dy, o)
        assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))


@pytest.mark.parametrize("T,G", [(5, 300), (1, 64), (70, 2000)])
def test_fewer_rows_than_groups(T, G):
    lens = [0] * G
    for r in range(T):
        lens[(r * 37 + 11) % G] += 1
    x, w, b, dy = data(T, G, 64, 40, torch.bfloat16, G)
    check(x, w, b, dy, edges(T, lens))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_starts(dtype):
    """rows and gradients that are slices of wider buffers, transposed, or start off the 16-byte grid; nothing outside them is read in"""
    T, K, N = 90, 40, 24
    o = edges(T, [50, 0, 33], 4)
    x, w, b, dy = data(T, 3, K, N, dtype, 3)
    y0, g0 = check(x, w, b, dy, o)
    for pad, start in ((8, 0), (8, 8), (3, 1), (0, 0)):
        wide = torch.full((T, K + pad + start), float("nan"), device="cuda", dtype=dtype)
        wide[:, start:start + K] = x
        wdy = torch.full((T, N + pad + start), float("nan"), device="cuda", dtype=dtype)
        wdy[:, start:start + N] = dy
        y, g = check(wide[:, start:start + K], w, b, wdy[:, start:start + N], o)
        assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))
    y, g = check(x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), b.t().contiguous().t(), dy, o)
    assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))
    one = x[:1]
    check(one.expand(T, K), w, b, dy, o)                                       # a broadcast row
    check(x, w, b, dy[:1].expand(T, N), o)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N", [(601, 523), (1031, 40), (44, 1543), (1030, 1030)])
def test_few_rows_that_begin_on_any_element(K, N, dtype):
    """rows and weights are read where they lie, forward and back: slices of wider buffers, whose rows start anywhere and end in what must not count"""
    T, G = 12, 3
    o = edges(T, [5, 0, 6], 1)
    x, w, b, dy = data(T, G, K, N, dtype, K)
    y0, g0 = check(x, w, b, dy, o)
    for pad, start in ((3, 1), (1, 0), (8, 5)):
        wide = torch.full((T, K + pad + start), float("nan"), device="cuda", dtype=dtype)
        wide[:, start:start + K] = x
        wdy = torch.full((T, N + pad + start), float("inf"), device="cuda", dtype=dtype)
        wdy[:, start:start + N] = dy
        ww = torch.full((G, N, K + pad + start), float("nan"), device="cuda", dtype=dtype)
        ww[:, :, start:start + K] = w
        y, g = check(wide[:, start:start + K], ww[:, :, start:start + K], b, wdy[:, start:start + N], o)
        assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))
    from uemda_amd.grouped import grouped_linear
    off, xl = torch.tensor(o, device="cuda"), x.clone().requires_grad_()      # the data gradient alone: dy is not copied either
    assert torch.equal(torch.autograd.grad(grouped_linear(xl, w, off, b), xl, wdy[:, start:start + N])[0], g0[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_group_and_of_other_groups_do_not_leak(dtype):
    from uemda_amd.grouped import grouped_linear
    T, K, N = 400, 72, 88
    o = edges(T, [130, 3, 140], 60)
    x, w, b, dy = data(T, 3, K, N, dtype, 4)
    x[:60], x[333:], dy[:60], dy[333:] = float("nan"), float("inf"), float("nan"), float("-inf")
    y, (dx, dw, db) = check(x.nan_to_num(0, 0, 0), w, b, dy.nan_to_num(0, 0, 0), o)
    off = torch.tensor(o, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    z = grouped_linear(*leaves[:2], off, leaves[2])
    gz = torch.autograd.grad(z, leaves, dy)
    assert torch.equal(z, y) and torch.equal(gz[0], dx) and torch.equal(gz[1], dw) and torch.equal(gz[2], db)
    assert not z[:60].any() and not z[333:].any() and not gz[0][:60].any() and not gz[0][333:].any()
    x[61, 5] = float("nan")                                                    # in group 0: its row of y, its group's dw, nothing else
    leaves[0] = x.clone().requires_grad_()
    z = grouped_linear(*leaves[:2], off, leaves[2])
    gz = torch.autograd.grad(z, leaves, dy)
    keep = torch.ones(T, dtype=torch.bool)
    keep[61] = False
    assert z[61].isnan().all() and torch.equal(z[keep], y[keep]) and torch.equal(gz[0], dx) and torch.equal(gz[1][1:], dw[1:])


@pytest.mark.parametrize("G", [3, 130])
def test_offsets_that_are_not_what_they_should_be(G):
    """any contents give disjoint groups inside the rows: entries are clamped to [0, rows] and to the largest in front of them"""
    T, K, N = 500, 32, 40
    g = torch.Generator().manual_seed(G)
    x, w, b, dy = data(T, G, K, N, torch.float32, 5)
    for trial in range(4):
        raw = torch.randint(-300, 900, (G + 1,), generator=g)
        if trial == 1:
            raw = raw * (2 ** 40)
        fixed = raw.clamp(0, T).cummax(0).values.tolist()
        from uemda_amd.grouped import grouped_linear
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = grouped_linear(leaves[0], leaves[1], raw.cuda(), leaves[2])
        gr = torch.autograd.grad(y, leaves, dy)
        y2, gr2 = check(x, w, b, dy, fixed)
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(gr, gr2))


def test_empty_rows_partial_gradients_and_the_module():
    from uemda_amd import UemError
    from uemda_amd.grouped import GroupedLinear, grouped_linear
    m = GroupedLinear(3, 16, 24).cuda()
    assert list(m.state_dict()) == ["weight", "bias"] and float(m.weight.abs().max()) <= 0.25
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    y = m(torch.empty(0, 16, device="cuda"), off)
    y.sum().backward()
    assert y.shape == (0, 24) and not m.weight.grad.any() and not m.bias.grad.any()
    x, w, b, dy = data(60, 3, 16, 24, torch.float32, 6)
    off = torch.tensor([0, 20, 20, 60], device="cuda")
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(grouped_linear(full[0], full[1], off, full[2]), full, dy)
    assert torch.equal(torch.autograd.grad(grouped_linear(full[0], w, off, b), full[0], dy)[0], gx)
    assert torch.equal(torch.autograd.grad(grouped_linear(x, full[1], off, b), full[1], dy)[0], gw)
    assert torch.equal(torch.autograd.grad(grouped_linear(x, w, off, full[2]), full[2], dy)[0], gb)
    with pytest.raises(UemError, match="gradient of the gradient"):
        torch.autograd.grad(grouped_linear(full[0], w, off).sum(), full[0], create_graph=True)


def test_gradient_against_differences():
    """y is linear in x, w and b: along a direction the difference is the derivative, and only the forward's rounding stands between"""
    from uemda_amd.grouped import grouped_linear
    T, K, N = 50, 24, 32
    o = edges(T, [20, 0, 25], 2)
    x, w, b, dy = data(T, 3, K, N, torch.float32, 7)
    _, (gx, gw, gb) = check(x, w, b, dy, o)
    off = torch.tensor(o, device="cuda")
    gen = torch.Generator().manual_seed(2)
    for i, (t, gr) in enumerate(((x, gx), (w, gw), (b, gb))):
        v = torch.randn(t.shape, generator=gen).sign().cuda()
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = t + v, t - v
        up, down = [grouped_linear(a[0], a[1], off, a[2]).double() for a in args]
        got = ((up - down) / 2 * dy.double()).sum()
        exact = (gr.double() * v.double()).sum()
        mags = sum((reference(a[0], a[1], a[2], dy, o)[0][1] * dy.double().abs()).sum() for a in args)
        moved = U * ((t.abs().double() + 1) * gr.double().abs()).sum()        # t + v and t - v round too
        assert abs(got - exact) <= U * (K + 9) * mags + 2 * moved + U * T * gr.double().abs().sum(), (i, float(got), float(exact))


def test_results_repeat_and_a_captured_step_takes_new_partitions():
    from uemda_amd.grouped import grouped_linear
    T, K, N, G = 3000, 256, 264, 5
    x, w, b, dy = data(T, G, K, N, torch.bfloat16, 8)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    off = torch.tensor([0, 600, 1300, 1300, 2900, 3000], dtype=torch.int32, device="cuda")

    def step():
        y = grouped_linear(leaves[0], leaves[1], off, leaves[2])
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    first = [t.clone() for t in step()]
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(step(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for o in ([0, 3000, 3000, 3000, 3000, 3000], [10, 20, 30, 40, 2000, 2001], [0, 0, 0, 0, 0, 3000]):
        off.copy_(torch.tensor(o, dtype=torch.int32))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want)), o


@pytest.mark.parametrize("K,N", [(48, 56), (33, 17), (600, 7)])
def test_master_weights_that_begin_on_any_element(K, N):
    """fp32 weights inside a flat parameter buffer, or the weights behind the first group, under bf16 rows: any 4-byte boundary"""
    o = edges(200, [60, 0, 100], 7)
    x, w, b, dy = data(200, 3, K, N, torch.bfloat16, 1, wdtype=torch.float32)
    y0, g0 = check(x, w, b, dy, o)
    for start in (1, 2, 3, 4):
        flat = torch.full((start + w.numel() + 5,), float("nan"), device="cuda")
        v = flat[start:start + w.numel()].view(3, N, K)
        v.copy_(w)
        assert v.is_contiguous()
        y, g = check(x, v, b, dy, o)
        assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))
    more = torch.cat([torch.full((1, N, K), float("nan"), device="cuda"), w])
    y, g = check(x, more[1:], b, dy, o)
    assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))


# T, K, N, lengths, rows in front; which of forward, data gradient, weight gradient run on tiles of 256 x 256 (the library is asked, so that a
# change of its rules cannot empty this).  A stage is 32 of the reduction: 1000 makes 32 stages (even), 776 and 777 make 25, 1001 makes 32
# with a ragged last one; the dominating groups are several chunks and a rest, whose partial sums are joined
LARGE = [
    (25000, 1000, 1000, [14001, 0, 5000, 3003, 1], 900, "fdw"),
    (28000, 776, 1000, [300, 20000, 257, 0, 5000], 31, "fdw"),
    (28000, 777, 1001, [0, 25111, 1, 255, 700], 1000, "fdw"),       # odd widths: padded copies, results element by element
    (28000, 1001, 777, [28000, 0, 0, 0, 0], 0, "fdw"),               # one group of all rows
    (28000, 1000, 1000, [0, 0, 0, 0, 0], 13, "fdw"),                 # no row has a group
    (30000, 1023, 1021, [5000, 5001, 4999, 5000, 5000, 4000], 500, "fdw"),
    (40000, 520, 1000, [39000, 1, 2, 3, 4, 500], 200, "fd"),
] + [(25000, k, 1000, [9000, 3, 0, 12000, 77], 5, "f") for k in (8, 33, 72, 104, 136, 168)] \
  + [(25000, 1000, n, [9000, 3, 0, 12000, 77], 5, "d") for n in (8, 33, 72, 104, 136, 168)]     # 1 to 6 stages: fewer than, as many as and more than the ring


@pytest.mark.parametrize("T,K,N,lens,head,forms", LARGE)
def test_tiles_of_256(T, K, N, lens, head, forms):
    from uemda_amd import _lib
    for form in forms:
        assert _lib.load().uem_grouped_tile_rows(T, len(lens), K, N, 1, "fdw".index(form)) == 256, form
    x, w, b, dy = data(T, len(lens), K, N, torch.bfloat16, T + K + N)
    o = edges(T, lens, head)
    x[:o[0]], dy[:o[0]], x[o[-1]:], dy[o[-1]:] = float("nan"), float("inf"), float("inf"), float("nan")      # rows of no group
    check(x, w, b, dy, o)


def test_tiles_of_256_repeat_to_the_bit():
    """both waves of a SIMD, the ring and the join in a fixed order: ten steps of the same operands, others between them"""
    from uemda_amd.grouped import grouped_linear
    T, K, N, lens = 28000, 776, 1000, [300, 20000, 257, 0, 5000]
    x, w, b, dy = data(T, 5, K, N, torch.bfloat16, 0)
    off = torch.tensor(edges(T, lens, 31), device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = grouped_linear(*leaves[:2], off, leaves[2])
        return y, *torch.autograd.grad(y, leaves, dy)
    want = once()
    for _ in range(9):
        grouped_linear(dy.detach(), w.detach().transpose(1, 2), off)
        assert all(torch.equal(p, q) for p, q in zip(once(), want))
