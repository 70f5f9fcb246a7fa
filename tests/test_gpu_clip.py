"""uemda_amd.optim.get_total_norm / clip_grad_norm_ over lists of tensors, against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def params_of(tensors):
    out = []
    for t in tensors:
        p = torch.empty(t.shape, device=t.device, dtype=t.dtype).requires_grad_()
        p.grad = t
        out.append(p)
    return out


def exact_norm(tensors, kind):
    flat = [t.double().flatten() for t in tensors if t.numel()]
    if not flat:
        return 0.0
    flat = torch.cat(flat)
    return float(flat.norm()) if kind == 2 else float(flat.abs().max())


def check(tensors, max_norm, kind=2):
    """in place: every element times min(max / (n + 1e-6), 1) in 32 bits.  n is the 64-bit norm rounded once (2^-24); the sum, the quotient
    and the product round once each: 4 half steps of fp32 for the coefficient and 1 for the product, and one of the type's own."""
    from uemda_amd.optim import clip_grad_norm_, get_total_norm
    before = [t.detach().clone() for t in tensors]
    want = exact_norm(before, kind)
    n0 = get_total_norm(tensors, kind if kind == 2 else INF)
    assert n0.shape == () and n0.dtype == torch.float32
    n = clip_grad_norm_(params_of(tensors), max_norm, kind if kind == 2 else INF)
    assert torch.equal(n, n0)
    assert abs(float(n) - want) <= 2.0 ** -23 * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for b, t in zip(before, tensors):
        if coef == 1.0 and max_norm > want * (1 + 1e-6) + 2e-6:
            assert torch.equal(b, t)
            continue
        ref = b.double() * coef
        tol = ref.abs() * (5 * 2.0 ** -24 + (torch.finfo(t.dtype).eps / 2 if t.dtype == torch.bfloat16 else 0)) + torch.finfo(t.dtype).tiny
        assert ((t.double() - ref).abs() <= tol).all()
    return n


def rand(g, n, dtype=torch.float32):
    return torch.randn(n, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("kind", [2, 0])
@pytest.mark.parametrize("sizes", [[1], [3], [4096], [1, 1, 1], [5, 1000, 17], [70001], [64] * 161, [9] * 500, [0, 7, 0], [2 ** 21 + 3, 5]])
def test_lists_of_one_type(sizes, kind):
    g = torch.Generator().manual_seed(sum(sizes) + len(sizes))
    for dtype in (torch.float32, torch.bfloat16):
        for max_norm in (0.5, 1e6, 0.0):
            check([rand(g, n, dtype) for n in sizes], max_norm, kind)


@pytest.mark.parametrize("seed", range(4))
def test_mixed_types_at_any_element_of_one_allocation(seed):
    """neighbours in one buffer: an access of 16 bytes may hold the ends of two or three tensors, and what is in no tensor stays as it was"""
    g = torch.Generator().manual_seed(seed)
    for dtype, guard in ((torch.float32, 7.0), (torch.bfloat16, 7.0)):
        flat = torch.full((60000,), guard, dtype=dtype).cuda()
        at, views, owned = 1 + seed, [], torch.zeros(60000, dtype=torch.bool)
        while True:
            n = int(torch.randint(1, 40, (1,), generator=g)) if torch.rand(1, generator=g) < 0.8 else int(torch.randint(1000, 20000, (1,), generator=g))
            if at + n > 59990:
                break
            views.append(flat[at:at + n])
            views[-1].copy_(torch.randn(n, generator=g).to(dtype))
            owned[at:at + n] = True
            at += n + int(torch.randint(0, 3, (1,), generator=g))
        others = [rand(g, 333, torch.float32), rand(g, 77, torch.bfloat16)]
        check(views + others, 1.0)
        assert (flat[~owned.cuda()] == guard).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tensor_of_more_than_2_to_the_31_elements(dtype):
    from uemda_amd.optim import clip_grad_norm_
    n = 2 ** 31 + 12345
    t = torch.zeros(n + 1, dtype=dtype, device="cuda")[1:]                     # off the 16-byte grid
    spots = [0, 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, n - 9, n - 1]
    for i, s in enumerate(spots):
        t[s] = 2.0 ** i
    want = math.sqrt(sum(4.0 ** i for i in range(len(spots))))
    got = clip_grad_norm_(params_of([t]), 1.0)
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    for i, s in enumerate(spots):                                              # 5 half steps of fp32, one of the type's
        ref = 2.0 ** i / (want + 1e-6)
        assert abs(float(t[s]) - ref) <= ref * (5 * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0))
    assert int(torch.count_nonzero(t)) == len(spots)


def test_layouts():
    from uemda_amd import UemError
    from uemda_amd.optim import clip_grad_norm_, get_total_norm
    g = torch.Generator().manual_seed(5)
    cl = torch.randn(8, 16, 3, 3, generator=g).cuda().contiguous(memory_format=torch.channels_last)
    tr = torch.randn(40, 30, generator=g).cuda().t()
    wide = torch.full((20, 50), 3.0).cuda()
    wide[:, :37] = torch.randn(20, 37, generator=g).cuda()
    check([cl, tr, wide[:, :37]], 1.0)
    assert (wide[:, 37:] == 3.0).all()
    row = torch.randn(1, 30, generator=g).cuda()
    assert abs(float(get_total_norm([row.expand(5, 30)])) - math.sqrt(5) * float(row.double().norm())) < 1e-5
    with pytest.raises(UemError, match="repeats"):
        clip_grad_norm_(params_of([row.expand(5, 30)]), 1.0)
    a = torch.randn(100, generator=g).cuda()
    with pytest.raises(UemError, match="share memory"):
        clip_grad_norm_(params_of([a, a]), 1.0)
    with pytest.raises(UemError, match="share memory"):
        clip_grad_norm_(params_of([a[:60], a[59:]]), 1.0)
    for pair in ([wide[:, :37], wide[:, :37]], [wide[:, :37], wide[:, 36:]], [wide[:, :37], wide[0, 30:40]]):      # with gaps: scaled in copies
        with pytest.raises(UemError, match="overlaps"):
            clip_grad_norm_(params_of(pair), 1.0)
    keep = a.clone()
    check([a[:60], a[60:]], 1.0)
    assert not torch.equal(a, keep)
    with pytest.raises(UemError, match="one MI355X device"):
        get_total_norm([a, a.cpu()])
    with pytest.raises(UemError, match="float32 or bfloat16"):
        get_total_norm([a.double()])


def test_skipped_and_single_parameters():
    from uemda_amd.optim import clip_grad_norm_
    a, b = torch.randn(9).cuda().requires_grad_(), torch.randn(9).cuda().requires_grad_()
    assert float(clip_grad_norm_([a, b], 1.0)) == 0.0
    b.grad = torch.full((9,), 2.0, device="cuda")
    assert float(clip_grad_norm_([a, b], 3.0)) == 6.0 and a.grad is None
    torch.testing.assert_close(b.grad, torch.full((9,), 1.0, device="cuda"), rtol=1e-6, atol=0)
    v = b.grad._version
    clip_grad_norm_(b, 0.3)
    assert b.grad._version > v                                                  # autograd sees the in-place change
    assert float(clip_grad_norm_([], 1.0)) == 0.0


@pytest.mark.parametrize("kind", [2, 0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_and_non_finite_values(kind, dtype):
    from uemda_amd.optim import clip_grad_norm_
    nt = 2 if kind == 2 else INF
    big = torch.full((1000,), 1e30, dtype=dtype).cuda()                         # squares leave 32 bits
    check([big], 1.0, kind)
    small = torch.full((1000,), 1e-30, dtype=dtype).cuda()
    n = clip_grad_norm_(params_of([small]), 1.0, nt)
    assert abs(float(n) / (float(small[0]) * (math.sqrt(1000) if kind == 2 else 1)) - 1) < 1e-6
    for bad in (float("nan"), INF, -INF):
        t, u = torch.ones(5000, dtype=dtype).cuda(), torch.ones(33, dtype=dtype).cuda()
        t[4321] = bad
        ref = [x.clone().float().requires_grad_() for x in (t, u)]
        for r, x in zip(ref, (t, u)):
            r.grad = x.float().clone()                                          # (a copy for fp32 too: torch scales it in place)
        want = torch.nn.utils.clip_grad_norm_(ref, 1.0, nt)
        got = clip_grad_norm_(params_of([t, u]), 1.0, nt)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        for r, x in zip(ref, (t, u)):
            assert torch.equal(x.float(), r.grad) or torch.equal(x.isnan(), r.grad.isnan()) and torch.equal(x.nan_to_num(0).float(), r.grad.nan_to_num(0))


def test_repeats_to_the_bit_and_replays_from_a_graph():
    from uemda_amd.optim import clip_grad_norm_
    g = torch.Generator().manual_seed(8)
    src = [rand(g, n, d) for n, d in ((300000, torch.float32), (77777, torch.bfloat16), (12, torch.float32))]
    work = [t.clone() for t in src]
    params = params_of(work)

    def once():
        for w, s in zip(work, src):
            w.copy_(s)
        return clip_grad_norm_(params, 2.0)
    n = once().clone()
    want = [w.clone() for w in work]
    for _ in range(3):
        assert torch.equal(once(), n) and all(torch.equal(w, x) for w, x in zip(work, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for k in range(3):
        with torch.no_grad():
            src[0].mul_(1.5)
        n = once().clone()
        want = [w.clone() for w in work]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, n) and all(torch.equal(w, x) for w, x in zip(work, want)), k


def test_a_model_arena_together_with_other_modules():
    """a model's parameters alone keep their arena path; with anything beside them the list is clipped as one"""
    from uemda_amd.models.Encoder import Deeplabv2
    from uemda_amd.norm import LayerNorm
    from uemda_amd.optim import clip_grad_norm_, grad_norm
    torch.manual_seed(0)
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True)).cuda()
    model.zero_grad()
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in model.parameters():
        p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    head = LayerNorm(2048).cuda()
    head.weight.grad, head.bias.grad = torch.randn(2048, device="cuda"), torch.randn(2048, device="cuda")
    alone = float(grad_norm(model)[0])
    both = math.hypot(alone, float(torch.cat([head.weight.grad, head.bias.grad]).double().norm()))
    before = [p.grad.clone() for p in list(model.parameters()) + list(head.parameters())]
    n = clip_grad_norm_(list(model.parameters()) + list(head.parameters()), 32.0)
    assert abs(float(n) / both - 1) < 1e-6
    for b, p in zip(before, list(model.parameters()) + list(head.parameters())):
        torch.testing.assert_close(p.grad, b * (32.0 / both), rtol=1e-6, atol=0)


def test_some_of_a_models_parameters_are_clipped_alone():
    """a single parameter, a list of some, the largest magnitude of all: only what is listed is measured and scaled; the list of all that is
    trained gives what the model's arena gives"""
    from uemda_amd.models.Encoder import Deeplabv2
    from uemda_amd.optim import clip_grad_norm_, grad_norm
    torch.manual_seed(0)
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True)).cuda()
    model.zero_grad()
    g = torch.Generator(device="cuda").manual_seed(1)
    params = list(model.parameters())

    def fill():
        for p in params:
            p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    for listed in (params[7], params[:1], params[3:90], params[1:]):
        fill()
        names = {id(p) for p in ([listed] if isinstance(listed, torch.Tensor) else listed)}
        before = [p.grad.clone() for p in params]
        want = exact_norm([b for b, p in zip(before, params) if id(p) in names], 2)
        n = clip_grad_norm_(listed, 0.5)
        assert abs(float(n) - want) <= 2.0 ** -23 * want
        for b, p in zip(before, params):                       # the coefficient and the product: 5 roundings of half a step
            ref = b.double() * (0.5 / (want + 1e-6)) if id(p) in names else b.double()
            assert ((p.grad.double() - ref).abs() <= ref.abs() * (5 * 2.0 ** -24 if id(p) in names else 0)).all()
    fill()
    before = [p.grad.clone() for p in params]
    want = exact_norm(before, 0)
    assert float(clip_grad_norm_(params, 0.5, INF)) == want
    for b, p in zip(before, params):
        ref = b.double() * (0.5 / (want + 1e-6))
        assert ((p.grad.double() - ref).abs() <= ref.abs() * (5 * 2.0 ** -24)).all()
    fill()
    before, alone = [p.grad.clone() for p in params], grad_norm(model)[0].clone()
    assert torch.equal(clip_grad_norm_(filter(lambda p: p.requires_grad, params), 32.0), alone)
    coef = torch.clamp(32.0 / (alone + 1e-6), max=1.0)
    for b, p in zip(before, params):
        assert torch.equal(p.grad, b * coef)


@pytest.mark.parametrize("kind", [2, INF])
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_a_norm_that_is_not_finite_raises_where_it_is_asked_to(kind, bad):
    """the signature of torch's two functions; nothing is scaled by a call that raises"""
    from uemda_amd import UemError
    from uemda_amd.models.Encoder import Deeplabv2
    from uemda_amd.optim import clip_grad_norm_, get_total_norm
    t, u = torch.full((5000,), 3.0).cuda(), torch.ones(33, dtype=torch.bfloat16).cuda()
    assert torch.equal(clip_grad_norm_(params_of([t.clone(), u.clone()]), 1.0, kind, True, foreach=False), get_total_norm([t, u], kind, error_if_nonfinite=True))
    assert float(clip_grad_norm_([], 1.0, error_if_nonfinite=True)) == float(get_total_norm([], error_if_nonfinite=True, foreach=True)) == 0.0
    t[77] = bad
    keep = [t.clone(), u.clone()]
    with pytest.raises(UemError, match="total norm is"):
        get_total_norm([t, u], kind, error_if_nonfinite=True)
    with pytest.raises(UemError, match="total norm is"):
        clip_grad_norm_(params_of([t, u]), 1.0, kind, error_if_nonfinite=True)
    assert torch.equal(t.nan_to_num(7.0), keep[0].nan_to_num(7.0)) and torch.equal(u, keep[1])
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True)).cuda()
    model.zero_grad()
    params = list(model.parameters())
    for p in params:
        p.grad.fill_(2.0)
    params[3].grad.view(-1)[0] = bad
    with pytest.raises(UemError, match="total norm is"):
        clip_grad_norm_(params, 1.0, kind, error_if_nonfinite=True)
    assert all(bool((p.grad == 2.0).all()) for p in params[4:])


def test_slots_of_parameters_without_a_gradient_do_not_count():
    """behind torch's zero_grad(set_to_none=True) the arena still holds the pass before: what no later pass has written is no gradient"""
    from uemda_amd.models.Encoder import Deeplabv2
    from uemda_amd.optim import clip_grad_norm_
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True)).cuda()
    model.zero_grad()
    params = list(model.parameters())
    for p in params:
        p.grad.fill_(1.0)
    for p in params[40:]:
        p.grad = None
    want = exact_norm([p.grad for p in params[:40]], 2)
    got = clip_grad_norm_(params, 1.0)
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    assert all(p.grad is None for p in params[40:])
    for p in params[:40]:
        assert ((p.grad.double() - 1 / (want + 1e-6)).abs() <= 5 * 2.0 ** -24 / want).all()
