"""Layer norm, grouped products and gradient clipping as one training step uses them: rows normalised, sent through the weights of their class,
gradients of everything clipped together -- against the same step in 64 bits, with the errors of each part carried on to the next."""
import pytest
import torch

from test_gpu_grouped import U, edges, reference as products
from test_gpu_layernorm import bounds, close, reference as norm

pytestmark = pytest.mark.gpu


def build(T, C, N, lens, seed, dtype=torch.float32):
    from uemda_amd.grouped import GroupedLinear
    from uemda_amd.norm import LayerNorm
    torch.manual_seed(seed)
    ln, gl = LayerNorm(C).cuda(), GroupedLinear(len(lens), C, N).cuda()
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5)
        ln.bias.uniform_(-0.5, 0.5)
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, C, generator=g) * 2 + 0.5).to(dtype).cuda()
    dy = torch.randn(T, N, generator=g).to(dtype).cuda()
    return ln, gl, x, dy


def step(ln, gl, x, dy, off, max_norm):
    from uemda_amd.optim import clip_grad_norm_
    params = list(ln.parameters()) + list(gl.parameters())
    for p in params:
        p.grad = None
    xl = x.detach().requires_grad_()
    y = gl(ln(xl), off)
    (y * dy).sum().backward()
    n = clip_grad_norm_(params + [xl], max_norm)
    return y.detach(), n, [p.grad for p in params], xl.grad


@pytest.mark.parametrize("T,C,N,lens,head", [(1, 40, 24, [1], 0), (300, 96, 72, [100, 0, 150], 20), (2000, 333, 77, [900, 1, 1000, 50], 9)])
def test_step_against_64_bits(T, C, N, lens, head):
    ln, gl, x, dy = build(T, C, N, lens, T)
    o = edges(T, lens, head)
    off = torch.tensor(o, dtype=torch.int32, device="cuda")
    y, n, grads, gx = step(ln, gl, x, dy, off, 1.0)
    w, b, W, B = (p.detach() for p in (ln.weight, ln.bias, gl.weight, gl.bias))
    # forward
    zero = torch.zeros_like(x)
    r = norm(x, w, b, zero, 1e-5)
    eh = bounds(x, zero, b, r)[0] + U * r[0].abs()                             # of the rows as stored
    h = r[0]
    (ry, ay), (rdh, adh), (rdW, adW), (rdB, adB) = products(h, W, B, dy, o)
    eW = products(eh, W.abs(), None, dy.abs(), o)                              # errors of h carried through |W| and |dy|
    close(y, ry, eW[0][0] + 2 * U * (C + 9) * ay, "y")
    # backward: dh of the products, then the norm's backward of it, the gradient itself being off by edh
    edh = 2 * U * (N + 8) * adh + U * rdh.abs()
    _, rdx, rdw, rdb, hat, rstd, g, w64 = norm(x, w, b, rdh, 1e-5)
    _, edx, edw, edb = bounds(x, rdh, b, norm(x, w, b, rdh, 1e-5))
    eg = edh * w64.abs()
    edx = edx + rstd * (eg + eg.mean(1, keepdim=True) + hat.abs() * (eg * hat.abs()).mean(1, keepdim=True))
    edw = edw + (edh * hat.abs()).sum(0)
    edb = edb + edh.sum(0)
    lens64 = torch.tensor(lens, dtype=torch.float64, device="cuda")
    edW = eW[2][0] + 2 * U * (lens64.view(-1, 1, 1) + 8) * adW
    edB = 2 * U * (lens64.view(-1, 1) + 8) * adB
    want, errs = [rdw, rdb, rdW, rdB, rdx], [edw, edb, edW, edB, edx]
    total = torch.sqrt(sum((t ** 2).sum() for t in want))
    err = torch.sqrt(sum((e ** 2).sum() for e in errs)) + 2 * U * total
    assert abs(float(n) - float(total)) <= float(err)
    coef = min(1.0, 1.0 / (float(total) + 1e-6))
    for name, got, t, e in zip(("dw", "db", "dW", "dB", "dx"), grads + [gx], want, errs):
        close(got, t * coef, e * coef + t.abs() * coef * (float(err) / float(total) + 5 * U), name)
    rows = torch.ones(T, dtype=torch.bool)
    rows[head:head + sum(lens)] = False
    assert not y[rows.cuda()].any() and not gx[rows.cuda()].any()              # rows of no class


def test_a_captured_step_of_all_three_replays_with_new_rows():
    """the step as one hipGraph: new rows, new partition, eager work and synchronisation between the replays"""
    from uemda_amd.optim import clip_grad_norm_
    T, C, N, lens = 1000, 128, 64, [400, 100, 450]
    ln, gl, x, dy = build(T, C, N, lens, 3, torch.bfloat16)
    params = list(ln.parameters()) + list(gl.parameters())
    off = torch.tensor(edges(T, lens, 10), device="cuda")

    def once():
        y = gl(ln(x), off)
        grads = torch.autograd.grad(y, params, dy)
        for p, g in zip(params, grads):
            p.grad = g
        return [y.detach(), clip_grad_norm_(params, 0.5)] + [p.grad for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    g = torch.Generator().manual_seed(9)
    for o in ([0, 500, 500, 1000], [1, 2, 3, 4], [100, 300, 900, 990]):
        x.copy_(torch.randn(T, C, generator=g).bfloat16())
        off.copy_(torch.tensor(o))
        want = [t.clone() for t in once()]
        for p in params:
            p.grad = None
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), o
