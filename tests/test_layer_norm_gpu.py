"""nn_helpers.layer_norm / LayerNorm on the GPU against the formulas in float64, element by element.

Tolerances (u = 2^-24, half a step of fp32).  A row's sum takes at most 32 additions per thread and 12 more between threads: N = 44
roundings, each of at most u of the terms' absolute sum.  So mean is off by N u mean|x|, the variance by (2 N + 4) u of itself plus
twice mean's error squared, and xhat by
    dxhat = rstd (N u mean|x| + 2 u |x|) + |xhat| (N + 6) u.
y adds two roundings; dx combines two more row sums with the same N; dw and db add rows one after another inside a workgroup (rows / 512
and 4 waves), then 32 + 16 partial rows.  Results in 16 bits add half a step of their type."""
import math

import pytest
import torch

from margipose_amd._lib import MposeError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
N = 44


def _half(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def _check(x, w, b, dy, eps, got):
    """x, dy (rows, cols) as given to the operator; got: y, dx, dw, db (None: not asked)."""
    x, dy = x.detach().double().cpu(), dy.detach().double().cpu()
    cols = x.shape[1]
    wd = torch.ones(cols, dtype=torch.float64) if w is None else w.detach().double().cpu().reshape(-1)
    bd = torch.zeros(cols, dtype=torch.float64) if b is None else b.detach().double().cpu().reshape(-1)
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xhat = (x - mean) * rstd
    dxh = rstd * (N * U * x.abs().mean(1, keepdim=True) + 2 * U * x.abs()) + xhat.abs() * (N + 6) * U
    dxh = dxh + xhat.abs() * rstd ** 2 * (N * U * x.abs().mean(1, keepdim=True)) ** 2
    y, dx, dw, db = got

    def close(name, a, want, tol, dtype):
        if a is None:
            return
        a = a.detach().double().cpu().reshape(want.shape)
        tol = tol + _half(dtype) * (want.abs() + tol) + (2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133)      # (a subnormal's half step)
        bad = ~((a - want).abs() <= tol)
        assert not bad.any(), (name, float(((a - want).abs() / tol).max()), int(bad.sum()))

    want = xhat * wd + bd
    close('y', y, want, wd.abs() * dxh + 2 * U * (want.abs() + (xhat * wd).abs()), y.dtype if y is not None else None)
    g = dy * wd
    mg, mgx = g.abs().mean(1, keepdim=True), (g * xhat).abs().mean(1, keepdim=True)
    m0, m1 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    want = rstd * (g - m0 - xhat * m1)
    e1 = (N + 2) * U * mgx + (g.abs() * dxh).mean(1, keepdim=True)
    tol = rstd * (2 * U * g.abs() + (N + 1) * U * mg + xhat.abs() * e1 + dxh * (m1.abs() + e1) + 4 * U * (g.abs() + m0.abs() + (xhat * m1).abs())) + (N + 6) * U * want.abs()
    close('dx', dx, want, tol, dx.dtype if dx is not None else None)
    chain = x.shape[0] / 512 + 4 + 48 + 2
    close('dw', dw, (dy * xhat).sum(0), (dy.abs() * dxh).sum(0) + chain * U * (dy * xhat).abs().sum(0), dw.dtype if dw is not None else None)
    close('db', db, dy.sum(0), chain * U * dy.abs().sum(0), db.dtype if db is not None else None)


def _inputs(rows, cols, dtype, seed, gap=0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols + gap, generator=g) * 2 + offset).to(dtype).cuda()[:, :cols]
    dy = torch.randn(rows, cols + gap, generator=g).to(dtype).cuda()[:, :cols]
    w = (1 + 0.3 * torch.randn(cols, generator=g)).cuda()
    b = (0.3 * torch.randn(cols, generator=g)).cuda()
    return x, w, b, dy


COLS = [1, 2, 3, 4, 63, 64, 65, 128, 255, 256, 257, 260, 512, 513, 1000, 1001, 1024, 1025, 1028, 2048, 2049, 4096, 4100, 8192, 8200, 16384, 16385, 20000]


@pytest.mark.parametrize('cols', COLS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_forward_and_backward_over_the_widths(cols, dtype):
    from margipose_amd.nn_helpers import layer_norm
    for rows, gap in ((1, 0), (5, 0), (131, 8), (130, 3)):
        x, w, b, dy = _inputs(rows, cols, dtype, cols + rows, gap)
        x.requires_grad_(True); w.requires_grad_(True); b.requires_grad_(True)
        y = layer_norm(x, (cols,), w, b)
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
        _check(x, w, b, dy, 1e-5, (y, dx, dw, db))
        with torch.no_grad():
            assert torch.equal(layer_norm(x, (cols,), w, b), y)


@pytest.mark.parametrize('rows,cols', [(2049, 64), (40000, 32), (8193, 1500), (3000, 3000), (700, 17000)])
def test_many_rows(rows, cols):
    from margipose_amd.nn_helpers import layer_norm
    x, w, b, dy = _inputs(rows, cols, torch.float32, rows)
    x.requires_grad_(True); w.requires_grad_(True); b.requires_grad_(True)
    y = layer_norm(x, (cols,), w, b)
    first = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    _check(x, w, b, dy, 1e-5, (y,) + first)
    again = torch.autograd.grad(y, (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_which_gradients_are_asked(dtype):
    from margipose_amd.nn_helpers import layer_norm
    for weight in (None, 'f32', 'own'):
        for bias in (False, True):
            for grads in ('x', 'w', 'xw'):
                x, w, b, dy = _inputs(33, 70, dtype, 7)
                w = None if weight is None else w if weight == 'f32' else w.to(dtype)
                b = None if not bias else b if weight != 'own' else b.to(dtype)
                x.requires_grad_('x' in grads)
                for t in (w, b):
                    if t is not None:
                        t.requires_grad_('w' in grads)
                leaves = [t for t in (x, w, b) if t is not None and t.requires_grad]
                y = layer_norm(x, 70, w, b, 1e-3)
                if not leaves:
                    assert not y.requires_grad
                    _check(x, w, b, dy, 1e-3, (y, None, None, None))
                    continue
                got = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
                _check(x, w, b, dy, 1e-3, (y, got.get(id(x)), got.get(id(w)) if w is not None else None, got.get(id(b)) if b is not None else None))
                assert w is None or id(w) not in got or got[id(w)].dtype == w.dtype


def test_shapes_strides_and_layouts():
    from margipose_amd.nn_helpers import layer_norm
    g = torch.Generator().manual_seed(3)
    base = torch.randn(4, 6, 5, 32, generator=g).cuda()
    w, b = torch.randn(32, generator=g).cuda(), torch.randn(32, generator=g).cuda()
    views = [base, base[:, ::2], base.transpose(0, 1), base.permute(1, 2, 0, 3), base[1:2], base[:, :1, :1].expand(4, 6, 5, 32), base[0, 0, 0],
             torch.randn(4, 32, 6, 5, generator=g).cuda().permute(0, 2, 3, 1),
             torch.randn(4, 32, 6, 5, generator=g).cuda().to(memory_format=torch.channels_last).permute(0, 2, 3, 1)]
    for v in views:
        x = v.detach().requires_grad_(True)
        y = layer_norm(x, (32,), w, b)
        for dy in (torch.randn(v.shape, generator=g).cuda(), torch.ones((), device='cuda').expand(v.shape), torch.randn(v.shape[::-1], generator=g).cuda().permute(*range(v.dim())[::-1])):
            (dx,) = torch.autograd.grad(y, (x,), dy, retain_graph=True)
            _check(x.reshape(-1, 32), w, b, dy.reshape(-1, 32), 1e-5, (y.reshape(-1, 32), dx.reshape(-1, 32), None, None))
    # several axes at once, weights of their shape
    w2, b2 = torch.randn(5, 32, generator=g).cuda().requires_grad_(True), torch.randn(5, 32, generator=g).cuda().requires_grad_(True)
    y = layer_norm(base, (5, 32), w2, b2)
    dw, db = torch.autograd.grad(y, (w2, b2), torch.ones_like(y))
    assert dw.shape == w2.shape and db.shape == b2.shape
    _check(base.reshape(-1, 160), w2, b2, torch.ones(24, 160), 1e-5, (y.reshape(-1, 160), None, dw, db))
    yb = layer_norm(base, (5, 32), None, b2)
    (db,) = torch.autograd.grad(yb, (b2,), torch.ones_like(y))
    assert db.shape == b2.shape
    # a broadcast leaf: its gradient is the sum over the copies
    leaf = torch.randn(32, generator=g).cuda().requires_grad_(True)
    layer_norm(leaf.expand(7, 32), (32,), w, b)[2].sum().backward()
    assert leaf.grad.shape == (32,)
    # no rows: empty results, zero gradients
    e = torch.zeros(0, 5, 32, device='cuda', requires_grad=True)
    we = w.clone().requires_grad_(True)
    y = layer_norm(e, (32,), we, b)
    de, dw = torch.autograd.grad(y, (e, we), torch.zeros_like(y))
    assert y.shape == de.shape == (0, 5, 32) and torch.equal(dw, torch.zeros_like(w))


def test_special_rows_stay_alone():
    from margipose_amd.nn_helpers import layer_norm
    for cols in (48, 1100, 17000):
        x, w, b, _ = _inputs(6, cols, torch.float32, 5)
        clean = layer_norm(x, (cols,), w, b)
        x = x.clone()
        x[1] = 3.25                                   # a constant row: xhat is zero
        x[2, 7] = float('nan')
        x[3, 0] = float('inf')
        x[4] *= 1e15
        y = layer_norm(x, (cols,), w, b)
        assert torch.equal(y[0], clean[0]) and torch.equal(y[5], clean[5])
        assert torch.equal(y[1], b)                   # (3.25 times a count below 2^20 is a whole number of fp32: the mean is exact)
        assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[4]).all()


def test_gradient_agrees_with_differences():
    """Central differences of the fp64 formula at the operator's inputs: step h leaves an error of h^2 |f'''| / 6 < 1e-7 of these values."""
    from margipose_amd.nn_helpers import layer_norm
    x, w, b, dy = _inputs(3, 9, torch.float32, 11)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(layer_norm(x, (9,), w, b), (x,), dy)
    xd, wd, bd, gd = (t.detach().double().cpu() for t in (x, w, b, dy))

    def f(v):
        m = v.mean(1, keepdim=True)
        return float((((v - m) / ((v - m).square().mean(1, keepdim=True) + 1e-5).sqrt() * wd + bd) * gd).sum())
    h = 1e-4
    for i in range(3):
        for j in range(9):
            p, q = xd.clone(), xd.clone()
            p[i, j] += h; q[i, j] -= h
            assert abs((f(p) - f(q)) / (2 * h) - float(dx[i, j])) < 2e-6


def test_module_streams_graphs_and_plans():
    from margipose_amd.nn_helpers import LayerNorm, init_parameters, layer_norm
    m = LayerNorm(40).cuda()
    ref = torch.nn.LayerNorm(40)
    assert list(m.state_dict()) == list(ref.state_dict())
    m.load_state_dict(ref.state_dict())
    with torch.no_grad():
        m.weight.fill_(2.0); m.bias.fill_(1.0)
    init_parameters(m)
    assert torch.equal(m.weight, torch.ones_like(m.weight)) and torch.equal(m.bias, torch.zeros_like(m.bias))
    assert LayerNorm(40, elementwise_affine=False).cuda()(torch.randn(3, 40, device='cuda')).shape == (3, 40)
    x = torch.randn(70, 40, device='cuda')
    side = torch.cuda.Stream()
    want = m(x).detach()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m(x).detach()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # forward and backward in a captured graph, replayed with other inputs between eager work
    xs, dy = x.clone().requires_grad_(True), torch.randn(70, 40, device='cuda')
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(m(xs), [xs] + list(m.parameters()), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(m(xs) * 1.5)                            # (the same leaves twice in one capture)
        grads = torch.autograd.grad(y, [xs] + list(m.parameters()), dy)
    for it in range(3):
        with torch.no_grad():
            xs.copy_(torch.randn(70, 40, device='cuda'))
        graph.replay()
        torch.cuda.synchronize()
        x2 = xs.detach().clone().requires_grad_(True)
        y2 = m(m(x2) * 1.5)
        g2 = torch.autograd.grad(y2, [x2] + list(m.parameters()), dy)
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(grads, g2)), it
    # a weight changed between forward and backward is refused by autograd
    y = layer_norm(xs, (40,), m.weight, m.bias)
    with torch.no_grad():
        m.weight.mul_(2.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    del y


def test_capture_over_leaves_of_a_live_eager_graph_is_refused():
    from margipose_amd.nn_helpers import LayerNorm
    m = LayerNorm(24).cuda()
    x = torch.randn(5, 24, device='cuda')
    y = m(x)                                          # an eager graph that holds the module's parameters
    with pytest.raises(MposeError, match='outside this capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            x.mul_(1.0)
            m(x)
    del y
    with torch.no_grad():
        m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = m(x)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(z, m(x))


def test_refusals():
    from margipose_amd.nn_helpers import layer_norm
    x, w = torch.randn(4, 8, device='cuda'), torch.randn(8, device='cuda')
    for args, match in (((x.double(), (8,)), 'float32, bfloat16 or float16'), ((x, (7,)), 'last axes'), ((x, ()), 'last axes'), ((x, (4, 8, 1)), 'last axes'),
                        ((x[:, :0], (0,)), 'no element'), ((x, (8,), w[:7]), 'weight must'), ((x, (8,), w.half()), 'weight must'), ((x, (8,), w.cpu()), 'weight must'),
                        ((x, (8,), None, w.cpu()), 'bias must'), ((x.half(), (8,), w.half(), w), 'one type'), ((x, (8,), w, None, -1.0), 'eps'),
                        ((x, (8,), w, None, math.inf), 'eps'), ((x, (8,), torch.randn(16, device='cuda')[::2]), 'contiguous')):
        with pytest.raises(MposeError, match=match):
            layer_norm(*args)
    x.requires_grad_(True)
    y = layer_norm(x, (8,), w)
    (dx,) = torch.autograd.grad(y.square().sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match='differentiated twice|once_differentiable|does not require grad'):
        dx.sum().backward()
