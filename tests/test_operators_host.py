"""What the operators refuse, on the CPU: nothing here launches a kernel."""
import pytest
import torch

from uemda_amd import _lib
from uemda_amd._lib import UemError


def test_layer_norm_refusals():
    from uemda_amd.norm import LayerNorm, layer_norm
    x = torch.zeros(4, 8)
    with pytest.raises(UemError, match="MI355X"):
        layer_norm(x)
    with pytest.raises(UemError, match="float32 or bfloat16"):
        layer_norm(x.half())
    with pytest.raises(UemError, match="must be a tensor"):
        layer_norm([1.0])
    with pytest.raises(UemError, match="channels"):
        LayerNorm(0)
    with pytest.raises(UemError, match="channel_dim"):
        LayerNorm(8, channel_dim=2)
    lib = _lib.load()
    assert lib.uem_layernorm_fwd(None, 8, None, None, None, None, None, 4, 8, 1e-5, 0, None) == -1
    assert lib.uem_layernorm_fwd(16, 7, None, None, 16, None, None, 4, 8, 1e-5, 0, None) == -1          # rows closer than their length
    assert lib.uem_layernorm_fwd(16, 8, None, None, 16, 16, None, 4, 8, 1e-5, 0, None) == -1            # mean without rstd
    assert lib.uem_layernorm_fwd(16, 8, None, None, 16, None, None, 0, 8, 1e-5, 0, None) == -1
    assert lib.uem_layernorm_fwd(16, 8, None, None, 16, None, None, 4, 8, 1e-5, 64, None) == -1
    assert lib.uem_layernorm_bwd(16, 8, 16, 8, None, 16, 16, 16, 16, None, None, 4, 8, 0, None) == -1     # gradients without a workspace
    assert b"workspace" in lib.uem_last_error()
    for rows, c in ((1, 5), (1000, 7), (10 ** 6, 256)):
        assert lib.uem_layernorm_workspace_floats(rows, c) >= 2 * c


def test_layer_norm_formula_against_differences():
    """the 64-bit formulas that the device tests hold the kernels to are each other's derivatives"""
    from test_gpu_layernorm import reference
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 7), (7,), (7,), (5, 7)))
    _, dx, dw, db = reference(x, w, b, dy, 1e-5)[:4]
    h = 1e-6
    for t, grad in ((x, dx), (w, dw), (b, db)):
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        t0 = t.clone()
        t.copy_(t0 + h * v); up = (reference(x, w, b, dy, 1e-5)[0] * dy).sum()
        t.copy_(t0 - h * v); down = (reference(x, w, b, dy, 1e-5)[0] * dy).sum()
        t.copy_(t0)
        assert abs((up - down) / (2 * h) - (grad * v).sum()) < 1e-7 * (1 + (grad * v).abs().sum())


def test_gradient_norm_refusals():
    from uemda_amd.optim import clip_grad_norm_, get_total_norm
    p = torch.ones(3, requires_grad=True)
    p.grad = torch.ones(3)
    with pytest.raises(UemError, match="MI355X"):
        get_total_norm([p.grad])
    with pytest.raises(UemError, match="MI355X"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(UemError, match="norm_type"):
        clip_grad_norm_([p], 1.0, norm_type=3)
    with pytest.raises(UemError, match="negative"):
        clip_grad_norm_([p], -1.0)
    with pytest.raises(UemError, match="negative"):
        clip_grad_norm_([p], float("nan"))
    with pytest.raises(UemError, match="expected tensors"):
        get_total_norm([1.0])
    with torch.inference_mode():
        frozen = torch.ones(3)
    p.grad = frozen
    with pytest.raises(UemError, match="inference"):
        clip_grad_norm_([p], 1.0)
    p.grad = torch.ones(3).to_sparse()
    with pytest.raises(UemError, match="dense"):
        clip_grad_norm_([p], 1.0)
    assert float(get_total_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    lib = _lib.load()
    from array import array
    ptrs, n = array("Q", [16, 20]), array("q", [2, 4])
    args = (ptrs.buffer_info()[0], n.buffer_info()[0])
    assert lib.uem_multi_clip(*args, b"\0\0", 2, 2, 16, 16, 1.0, None) == -1 and b"share memory" in lib.uem_last_error()
    assert lib.uem_multi_norm(*args, b"\0\0", 2, 3, 16, 16, None) == -1 and b"norm type" in lib.uem_last_error()
    assert lib.uem_multi_norm(*args, b"\0\0", -1, 2, 16, 16, None) == -1
    ptrs[0] = 18
    assert lib.uem_multi_norm(*args, b"\0\0", 2, 2, 16, 16, None) == -1 and b"element boundary" in lib.uem_last_error()
    ptrs[0] = 0
    assert lib.uem_multi_norm(*args, b"\0\0", 2, 2, 16, 16, None) == -1
    assert lib.uem_multi_norm_workspace_doubles(3) == _lib.UEM_MULTI_BLOCKS + 6


def test_grouped_linear_refusals():
    from uemda_amd.grouped import GroupedLinear, grouped_linear
    x, w, off = torch.zeros(6, 8), torch.zeros(2, 4, 8), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(UemError, match="MI355X"):
        grouped_linear(x, w, off)
    for bad, text in (((x[0], w, off), "expected x"), ((x, w[0], off), "expected x"), ((x, torch.zeros(2, 4, 9), off), "expected x"),
                      ((x, torch.zeros(0, 4, 8), off), "expected x"), ((x.half(), w.half(), off), "float32"),
                      ((x, w.bfloat16(), off), "float32"), ((x, w, off[:2]), "offsets"), ((x, w, off.float()), "offsets"),
                      ((x, w, off, torch.zeros(2, 5)), "bias"), ((x, w, off, torch.zeros(2, 4).half()), "bias"), ((x, w, [0, 1, 2]), "tensor")):
        with pytest.raises(UemError, match=text):
            grouped_linear(*bad)
    with pytest.raises(UemError, match="positive"):
        GroupedLinear(0, 8, 8)
    lib = _lib.load()
    assert lib.uem_grouped_fwd(None, 8, 16, 8, None, 16, 16, 4, 2, 8, 8, 0, None) == -1
    assert lib.uem_grouped_fwd(16, 6, 16, 8, None, 16, 16, 4, 2, 6, 8, 0, None) == -1 and b"16-byte" in lib.uem_last_error()
    assert lib.uem_grouped_any_rows(4, 2, 6, 8, 0, 0) == 0 and lib.uem_grouped_any_rows(4, 2, 600, 8, 0, 0) == 1          # few rows, long ones
    assert lib.uem_grouped_any_rows(4, 2, 600, 8, 0, 1) == 0 and lib.uem_grouped_any_rows(4, 2, 8, 600, 0, 1) == 1
    assert lib.uem_grouped_any_rows(10 ** 6, 2, 600, 8, 0, 0) == 0
    assert lib.uem_grouped_fwd(18, 600, 16, 600, None, 16, 16, 4, 2, 600, 8, 0, None) == -1 and b"element" in lib.uem_last_error()
    assert lib.uem_grouped_fwd(24, 8, 16, 8, None, 16, 16, 4, 2, 8, 8, 0, None) == -1
    assert lib.uem_grouped_fwd(16, 4, 16, 8, None, 16, 16, 4, 2, 8, 8, 0, None) == -1 and b"shorter" in lib.uem_last_error()
    assert lib.uem_grouped_fwd(16, 8, 16, 8, None, 16, 16, 1 << 30, 2, 8, 8, 0, None) == -1
    assert lib.uem_grouped_dgrad(16, 8, 16, 8, 16, 16, 4, 2, 8, 8, 64, None) == -1
    assert lib.uem_grouped_wgrad(16, 8, 16, 8, None, 16, 16, 16, 4, 2, 8, 8, 0, None) == -1
    assert lib.uem_grouped_wgrad(16, 8, 16, 8, 16, 16, None, 16, 1 << 20, 2, 8, 8, 0, None) == -1 and b"workspace" in lib.uem_last_error()
    assert lib.uem_grouped_pad(16, 4, 16, 8, 6, 4, 0, None) == -1
    for T, G, K, N in ((1, 1, 1, 1), (100, 3, 5, 7), (1 << 20, 64, 2048, 2048), (1 << 20, 2, 8, 8)):
        assert lib.uem_grouped_wgrad_workspace_floats(T, G, K, N, 0) >= (0 if T < 1000 else N * (K + 1))


def test_the_host_extension_needs_its_binding():
    import subprocess
    import sys
    code = "import torch\nfrom uemda_amd import _host\ntry:\n    _host.layer_norm(torch.zeros(2, 8), None, None, 1e-5)\nexcept RuntimeError as e:\n    assert 'bound' in str(e)\nelse:\n    raise SystemExit(1)"
    assert subprocess.run([sys.executable, "-c", code]).returncode == 0


def test_only_a_whole_model_takes_its_arena(monkeypatch):
    """a model's arena is clipped where the list is all that the model trains; some of its parameters are a list like any other"""
    from uemda_amd import optim

    class Model(torch.nn.Linear):
        def flat_parameters(self):
            raise LookupError("arena")
    lists = []
    monkeypatch.setattr(_lib, "host", lambda: type("host", (), {"multi_norm": staticmethod(lambda ps, *a: lists.append(ps) or torch.tensor(1.0))}))
    m, other = Model(3, 2), torch.ones(2, requires_grad=True)
    for p in m.parameters():
        p._uem_owner, p.grad = m, torch.ones_like(p)
    w, b = m.parameters()
    for some in (w, [w], [b], [w, b, other], iter([b])):
        assert float(optim.clip_grad_norm_(some, 1.0)) == 1.0
    assert [len(ps) for ps in lists] == [1, 1, 1, 3, 1] and lists[0][0] is w and lists[4][0] is b
    assert float(optim.clip_grad_norm_([w, b], 1.0, float("inf"))) == 1.0 and len(lists) == 6
    b.requires_grad_(False)
    optim.clip_grad_norm_([w], 1.0)                            # b is frozen, but what it holds is no gradient of the list
    assert len(lists) == 7
    b.grad = None
    for whole in ([w], [w, b], m.parameters(), filter(lambda p: p.requires_grad, m.parameters())):
        with pytest.raises(LookupError, match="arena"):
            optim.clip_grad_norm_(whole, 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(UemError, match="negative"):
            optim.clip_grad_norm_([w, b], bad)
    assert len(lists) == 7


def test_forward_mode_and_traces_are_refused():
    """a call without requires_grad does not reach the autograd node: nothing but the operator itself can see a tangent that it would drop"""
    import torch.autograd.forward_ad as fa

    from uemda_amd.grouped import grouped_linear
    from uemda_amd.norm import layer_norm
    from uemda_amd.optim import clip_grad_norm_, get_total_norm
    x, w, b = torch.ones(6, 8), torch.ones(8), torch.zeros(8)
    gw, gb, off = torch.ones(2, 4, 8), torch.zeros(2, 4), torch.tensor([0, 3, 6])
    p = torch.ones(3, requires_grad=True)
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))
        p.grad = dual(torch.ones(3))
        calls = [lambda: layer_norm(dual(x), w, b), lambda: layer_norm(x, dual(w), b), lambda: layer_norm(x, w, dual(b)), lambda: layer_norm(dual(x)),
                 lambda: grouped_linear(dual(x), gw, off, gb), lambda: grouped_linear(x, dual(gw), off), lambda: grouped_linear(x, gw, off, dual(gb)),
                 lambda: get_total_norm([dual(w)]), lambda: clip_grad_norm_([p], 1.0)]
        for k, call in enumerate(calls):
            with pytest.raises(UemError, match="forward-mode"):
                call()
                pytest.fail(str(k))
    p.grad = None
    for fn, args in ((layer_norm, (x,)), (lambda a: layer_norm(a, w, b), (x,)), (grouped_linear, (x, gw, off)), (lambda a: get_total_norm([a]), (x,))):
        with pytest.raises(UemError, match="traced"):
            torch.jit.trace(fn, args)


def test_sums_over_ranks_are_not_clipped_together_with_other_gradients(monkeypatch):
    """behind reduce_gradients a model's arena holds sums, until it is cleared, its gradients are dropped or FusedSGD.step has averaged them"""
    from uemda_amd import dp, optim

    class Model(torch.nn.Linear):
        def flat_parameters(self):
            return torch.zeros(8), torch.zeros(8), 8
    lists = []
    monkeypatch.setattr(_lib, "host", lambda: type("host", (), {"multi_norm": staticmethod(lambda ps, *a: lists.append(ps) or torch.tensor(1.0))}))
    monkeypatch.setattr(dp, "world_size", lambda: 2)
    monkeypatch.setattr(dp.dist, "broadcast", lambda *a, **k: None)
    monkeypatch.setattr(dp.dist, "all_reduce", lambda *a, **k: None)
    monkeypatch.setattr(optim, "call", lambda *a: None)
    monkeypatch.setattr(optim, "stream", lambda: None)
    m, other, bare = Model(3, 2), torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True)
    for i, p in enumerate(m.parameters()):
        p._uem_owner, p._uem_off = m, 4 * i
    both = [*m.parameters(), other]

    def gradients():
        for p in both:
            p.grad = torch.ones_like(p)
    gradients()
    wrap = dp.DataParallel(m, overlap=False)
    optim.clip_grad_norm_(both, 1.0)
    assert wrap.reduce_gradients() == 0.5
    with pytest.raises(UemError, match="sums over ranks"):
        optim.clip_grad_norm_(both, 1.0)
    with pytest.raises(UemError, match="sums over ranks"):
        optim.clip_grad_norm_([other, m.bias], 1.0, float("inf"))
    optim.clip_grad_norm_([other], 1.0)
    optim.clip_grad_norm_([m.bias, bare], 1.0)                 # (bare has no gradient: one scale)
    assert len(lists) == 3
    optim.FusedSGD(m).step(max_norm=None, grad_prescale=0.5)
    optim.clip_grad_norm_(both, 1.0)
    wrap.reduce_gradients()
    with pytest.raises(UemError, match="sums over ranks"):
        optim.clip_grad_norm_(both, 1.0)
    gradients()                                                # new ones, as behind zero_grad(set_to_none=True)
    optim.clip_grad_norm_(both, 1.0)
    monkeypatch.setattr(dp, "world_size", lambda: 1)
    dp.DataParallel(m, overlap=False).reduce_gradients()       # a single rank's sum is its average
    optim.clip_grad_norm_(both, 1.0)
    assert len(lists) == 6


def test_clearing_a_models_gradients_ends_their_being_sums(monkeypatch):
    from uemda_amd import dp, optim
    from uemda_amd.models.Encoder import Deeplabv2
    monkeypatch.setattr(dp, "world_size", lambda: 2)
    monkeypatch.setattr(dp.dist, "broadcast", lambda *a, **k: None)
    monkeypatch.setattr(dp.dist, "all_reduce", lambda *a, **k: None)
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True))
    model._flatten_parameters()
    model.zero_grad()
    dp.DataParallel(model, overlap=False).reduce_gradients()
    assert optim._holds_sums(model)
    model.zero_grad()
    assert not optim._holds_sums(model)


def test_more_tiles_than_a_launch_has_threads_for_are_refused():
    """allowed sizes whose tiles, at 256 or 512 threads each, do not fit the 2^32 threads of a launch: said so before anything is launched"""
    lib = _lib.load()
    many, wide = 65535, 65536
    for flags in (0, 1):
        assert lib.uem_grouped_fwd(16, 8, 16, 8, None, 16, 16, many, many, 8, wide, flags, None) == -1 and b"2^32 threads" in lib.uem_last_error()
        assert lib.uem_grouped_dgrad(16, 8, 16, wide, 16, 16, many, many, wide, 8, flags, None) == -1 and b"2^32 threads" in lib.uem_last_error()
        assert lib.uem_grouped_wgrad(16, wide, 16, 8, 16, 16, 16, 16, many, many, 8, wide, flags, None) == -1 and b"2^32 threads" in lib.uem_last_error()


def test_the_tile_that_sizes_are_cut_into():
    lib = _lib.load()
    assert [lib.uem_grouped_tile_rows(32768, 7, 2048, 512, 1, form) for form in range(3)] == [128, 256, 256]
    assert lib.uem_grouped_tile_rows(9, 6, 2048, 512, 1, 0) == 32 and lib.uem_grouped_tile_rows(9, 6, 512, 2048, 1, 1) == 32      # few rows, long reductions
    assert lib.uem_grouped_tile_rows(9, 6, 2048, 512, 1, 1) == 64      # 256 tiles of 32 x 32 are too many for a reduction of 512
    for args in ((0, 1, 8, 8, 1, 0), (8, 1, 8, 8, 1, 3), (8, 1, 8, 8, 1, -1)):
        assert lib.uem_grouped_tile_rows(*args) == -1


def test_a_models_arena_is_its_gradients_only_where_they_are_its_slots():
    """a parameter without a gradient, or with a tensor of the caller's, leaves its slot of the arena with something else in it"""
    from uemda_amd import optim
    from uemda_amd.models.Encoder import Deeplabv2
    model = Deeplabv2(dict(backbone=dict(resnet_type="resnet50", output_stride=16, pretrained=False), multi_layer=True, cascade=False, use_ppm=False,
                           ppm=dict(num_classes=6, use_aux=False, fc_dim=2048), inchannels=2048, num_classes=6, is_ins_norm=True))
    model._flatten_parameters()
    params = list(model.parameters())
    assert optim._arena_of(params) is None                     # no gradient yet
    model.zero_grad()
    assert optim._arena_of(params) is model and optim._arena_of(params[1:]) is None
    slot, params[5].grad = params[5].grad, None
    assert optim._arena_of(params) is None
    params[5].grad = torch.zeros_like(params[5])
    assert optim._arena_of(params) is None
    params[5].grad = slot
    params[9].requires_grad_(False)
    params[9].grad = None
    assert optim._arena_of(params) is model and optim._arena_of([p for p in params if p.requires_grad]) is model
