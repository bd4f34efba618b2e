"""Cases for the training operators: orthogonalised updates (Newton-Schulz), the Muon and AdamW optimiser steps, layer normalisation.

`own` False: the operators in plain torch operations (float32, float64 where 32 bits lose what matters).  `own` True: the calls a user
makes of margipose_amd.  Both run the same inputs: `prepare` makes them from the seed, `run` is one pass and returns everything it computes.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)          # x -> a x + b x^3 + c x^5 on the singular values, five times
STEPS = 5
NS_EPS = 1e-7
MUON = {'lr': 0.02, 'momentum': 0.95, 'weight_decay': 0.01}
ADAMW = {'lr': 0.002, 'momentum': 0.9, 'beta2': 0.999, 'eps': 1e-8, 'weight_decay': 0.01}
ADAMW_STEPS_BEFORE = 9
LN_EPS = 1e-5

# The weights of one heat-map column and of the default model (four stages, twelve columns, InceptionV4 features), flattened to
# (leading dimension, the rest); and the lengths of the model's batch-norm vectors.
COLUMN = '9*192x1728,2*192x1152,4*192x192,2*192x128,7*128x1152,3*128x128,17x1152,17x128,17x153'
MODEL = ('109*192x1728,84*128x1152,48*192x192,36*128x128,24*192x1152,24*192x128,12*17x1152,12*17x128,12*17x153,5*96x576,3*128x51,'
         '2*64x160,2*64x384,2*64x448,2*96x384,128x384,32x27,32x288,64x288,96x864')
MODEL_VECTORS = '362*192,291*128,72*17,16*96,14*64,4*32'


def listed():
    return [
        # the twelve heat-map heads of the default model, alone: many tiny matrices, latency counts
        {'name': 'orth_heads', 'op': 'orth', 'shapes': '12*17x128', 'dtype': 'float32'},
        # an odd collection in half precision: single rows and columns, both orientations, sizes next to a tile's edge
        {'name': 'orth_ragged', 'op': 'orth', 'shapes': '1x64,64x1,33x31,130x51,65x257,1000x333,2*129x640,255x255', 'dtype': 'float16'},
        # one wide projection in bfloat16: few output tiles, long sums
        {'name': 'orth_wide', 'op': 'orth', 'shapes': '1024x4096', 'dtype': 'bfloat16'},
        # the largest square matrix
        {'name': 'orth_square', 'op': 'orth', 'shapes': '4096x4096', 'dtype': 'float32'},
        # a training step that fine-tunes one column: its matrices by Muon, its norms by AdamW
        {'name': 'muon_column', 'op': 'muon', 'shapes': COLUMN, 'vectors': '26*192,18*128,6*17'},
        # a training step of the default model, every parameter of it
        {'name': 'muon_model', 'op': 'muon', 'shapes': MODEL, 'vectors': MODEL_VECTORS},
        # the norm vectors of one stage's three columns
        {'name': 'adamw_norms', 'op': 'adamw', 'shapes': '78*192,54*128,18*17'},
        # every parameter of the default model by AdamW
        {'name': 'adamw_model', 'op': 'adamw', 'shapes': MODEL + ',' + MODEL_VECTORS},
        # one skeleton's 17 joint tokens, inference
        {'name': 'norm_joints', 'op': 'norm', 'rows': 17, 'cols': 128, 'gap': 0, 'dtype': 'float32', 'train': False},
        # the 32x32 feature map of a batch of 32 over its 128 channels, training
        {'name': 'norm_map', 'op': 'norm', 'rows': 32768, 'cols': 128, 'gap': 0, 'dtype': 'float32', 'train': True},
        # an odd width in half precision, rows apart from each other, training
        {'name': 'norm_odd', 'op': 'norm', 'rows': 4099, 'cols': 1001, 'gap': 23, 'dtype': 'float16', 'train': True},
        # wide tokens of a long batch in bfloat16, training
        {'name': 'norm_wide', 'op': 'norm', 'rows': 32768, 'cols': 4096, 'gap': 0, 'dtype': 'bfloat16', 'train': True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['orth', 'orth', 'muon', 'adamw', 'norm', 'norm'])
    if op == 'norm':
        cols = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, max(2, min(262144, (1 << 27) // cols)))
        return {'op': 'norm', 'rows': rows, 'cols': cols, 'gap': rng.choice([0, 0, 0, 8, 5]), 'dtype': rng.choice(['float32', 'bfloat16', 'float16']),
                'train': rng.random() < 0.7}
    if op == 'adamw':
        shapes = ['%d*%d' % (_spread(rng, 1, 100), _spread(rng, 1, 400000)) for _ in range(rng.randint(1, 4))]
        return {'op': 'adamw', 'shapes': ','.join(shapes)}
    if op == 'orth' and rng.random() < 0.4:
        m, n = _spread(rng, 64, 4096), _spread(rng, 64, 4096)
        return {'op': 'orth', 'shapes': '%dx%d' % (m, n), 'dtype': rng.choice(['float32', 'bfloat16', 'float16'])}
    shapes = ['%d*%dx%d' % (rng.randint(1, 6), _spread(rng, 1, 512), _spread(rng, 1, 2304)) for _ in range(rng.randint(1, 6))]
    if op == 'orth':
        return {'op': 'orth', 'shapes': ','.join(shapes), 'dtype': rng.choice(['float32', 'bfloat16', 'float16'])}
    return {'op': 'muon', 'shapes': ','.join(shapes), 'vectors': '%d*%d,%d*%d' % (rng.randint(1, 200), _spread(rng, 1, 512), rng.randint(1, 8), _spread(rng, 1, 4096))}


def _shapes(text):
    """'2*17x128,5' -> [(2, (17, 128)), (1, (5,))]."""
    parts = [p.split('*') if '*' in p else ('1', p) for p in text.split(',') if p]
    return [(int(k), tuple(int(s) for s in dims.split('x'))) for k, dims in parts]


def _stride(dims):
    return (math.prod(dims) + 3) // 4 * 4            # parameters lie in one arena, each at a multiple of 16 bytes


def _groups(flat, text):
    """The arena's parameters as one (count, *dims) tensor for each entry of `text`."""
    out, at = [], 0
    for k, dims in _shapes(text):
        n = k * _stride(dims)
        out.append(flat[at:at + n].view(k, _stride(dims))[:, :math.prod(dims)].unflatten(1, dims))
        at += n
    return out


def _arena(text, device):
    return torch.zeros(sum(k * _stride(dims) for k, dims in _shapes(text)), device=device)


def _gradients(k, m, n, gen):
    """Sums of outer products of output gradients and rectified activations, as a layer's weight gradient is."""
    s = 2 * min(m, n) + 8
    dev = gen.device
    a = torch.randn(k, m, s, generator=gen, device=dev)
    b = torch.randn(k, s, n, generator=gen, device=dev).relu_()
    return torch.matmul(a, b) * (0.05 / math.sqrt(s))


def _fill(flat, text, gen, gradients):
    for v in _groups(flat, text):
        if v.dim() == 3 and gradients:
            v.copy_(_gradients(*v.shape, gen))
        else:
            v.copy_(torch.randn(v.shape, generator=gen, device=gen.device) * (1e-3 if gradients else math.sqrt(2.0 / v.shape[-1])))


def _tensors(flat, text):
    return [t for v in _groups(flat, text) for t in v.unbind(0)]


def _gather(tensors, text):
    """Separate tensors, laid out like the arena of their parameters."""
    flat, at = _arena(text, 'cuda'), 0
    for v in _groups(flat, text):
        v.copy_(torch.stack(tensors[at:at + len(v)]))
        at += len(v)
    return flat


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    s = {'case': case}
    if case['op'] == 'norm':
        dtype = getattr(torch, case['dtype'])
        rows, cols = case['rows'], case['cols']
        x = torch.randn(rows, cols + case['gap'], generator=gen, device='cuda') * (0.5 + torch.rand(rows, 1, generator=gen, device='cuda'))
        s['x'] = (x + 0.5 * torch.randn(cols + case['gap'], generator=gen, device='cuda')).to(dtype)[:, :cols]
        s['weight'] = 1.0 + 0.2 * torch.randn(cols, generator=gen, device='cuda')
        s['bias'] = 0.2 * torch.randn(cols, generator=gen, device='cuda')
        if case['train']:
            s['dy'] = (0.1 * torch.randn(rows, cols, generator=gen, device='cuda')).to(dtype)
            for t in (s['x'], s['weight'], s['bias']):
                t.requires_grad_(True)
        return s
    if case['op'] == 'orth':
        dtype = getattr(torch, case['dtype'])
        s['groups'] = [_gradients(k, *dims, gen).to(dtype) for k, dims in _shapes(case['shapes'])]
        s['matrices'] = [t for g in s['groups'] for t in g.unbind(0)]
        return s
    matrices, vectors = (case['shapes'], case['vectors']) if case['op'] == 'muon' else ('', case['shapes'])
    s['texts'] = (matrices, vectors)
    for name, text in (('m', matrices), ('v', vectors)):
        s['p' + name], g = _arena(text, 'cuda'), _arena(text, 'cuda')
        _fill(s['p' + name], text, gen, False)
        _fill(g, text, gen, True)
        s['g' + name] = [t.clone() for t in _tensors(g, text)]          # the backward pass leaves a tensor for each parameter
    s['momentum'] = _arena(matrices, 'cuda')
    _fill(s['momentum'], matrices, gen, True)
    s['momentum'] *= 8.0
    s['exp_avg'], s['exp_avg_sq'] = _arena(vectors, 'cuda'), _arena(vectors, 'cuda')
    _fill(s['exp_avg'], vectors, gen, True)
    _fill(s['exp_avg_sq'], vectors, gen, True)
    s['exp_avg_sq'].square_()
    s['steps'] = ADAMW_STEPS_BEFORE
    if own:          # the optimiser that a training loop keeps, in the state that it has after some steps
        from margipose_amd.train_helpers import DeviceAdamW, DeviceMuon
        pm, pv = ([torch.nn.Parameter(t) for t in _tensors(s['p' + k], text)] for k, text in (('m', matrices), ('v', vectors)))
        for p, g in zip(pm + pv, s['gm'] + s['gv']):
            p.grad = g
        adamw = {'lr': ADAMW['lr'], 'betas': (ADAMW['momentum'], ADAMW['beta2']), 'eps': ADAMW['eps'], 'weight_decay': ADAMW['weight_decay']}
        if case['op'] == 'muon':
            opt = DeviceMuon(pm, vectors=pv, ns_steps=STEPS, ns_coefficients=COEFFICIENTS, ns_eps=NS_EPS, vector_options=adamw, **MUON)
            opt.momentum_arena.copy_(s['momentum'])
            s['momentum'] = opt.momentum_arena
        else:
            opt = DeviceAdamW(pv, **adamw)
        opt.exp_avg_arena.copy_(s['exp_avg'])
        opt.exp_avg_sq_arena.copy_(s['exp_avg_sq'])
        opt.steps = ADAMW_STEPS_BEFORE
        s['exp_avg'], s['exp_avg_sq'], s['optimiser'] = opt.exp_avg_arena, opt.exp_avg_sq_arena, opt
    return s


def _newton_schulz(g):
    """(k, m, n) -> the polynomial of the normalised matrices' singular values, in float32."""
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.mT.contiguous()
    x = x / (x.double().square().sum((1, 2), keepdim=True).sqrt() + NS_EPS).float()
    for _ in range(STEPS):
        s = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.mT if tall else x


def _plain_muon(s):
    h = MUON
    g = _gather(s['gm'], s['texts'][0])
    s['momentum'].mul_(h['momentum']).add_(g)
    u = g + h['momentum'] * s['momentum']
    for p, v in zip(_groups(s['pm'], s['texts'][0]), _groups(u, s['texts'][0])):
        scale = 0.2 * math.sqrt(max(p.shape[1:]))
        p.mul_(1.0 - h['lr'] * h['weight_decay']).sub_(h['lr'] * scale * _newton_schulz(v))


def _plain_adamw(s):
    h = ADAMW
    g = _gather(s['gv'], s['texts'][1])
    s['steps'] += 1
    b1, b2, t = h['momentum'], h['beta2'], s['steps']
    s['exp_avg'].mul_(b1).add_((1.0 - b1) * g)
    s['exp_avg_sq'].mul_(b2).add_((1.0 - b2) * g.square())
    denominator = (s['exp_avg_sq'] / (1.0 - b2 ** t)).sqrt() + h['eps']
    s['pv'].mul_(1.0 - h['lr'] * h['weight_decay']).sub_(h['lr'] / (1.0 - b1 ** t) * s['exp_avg'] / denominator)


def _plain_norm(s):
    with torch.no_grad():
        x, w = s['x'].float(), s['weight']
        centred = x - x.mean(1, keepdim=True)
        rstd = 1.0 / (centred.square().mean(1, keepdim=True) + LN_EPS).sqrt()
        xhat = centred * rstd
        y = (xhat * w + s['bias']).to(s['x'].dtype)
        if 'dy' not in s:
            return {'y': y}
        dy = s['dy'].float()
        g = dy * w
        dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * rstd
        return {'y': y, 'dx': dx.to(s['x'].dtype), 'dweight': (dy * xhat).sum(0), 'dbias': dy.sum(0)}


def run(state):
    op = state['case']['op']
    if op == 'norm':
        if not own:
            return _plain_norm(state)
        from margipose_amd.nn_helpers import layer_norm
        x, w, b = state['x'], state['weight'], state['bias']
        y = layer_norm(x, (x.shape[1],), w, b, LN_EPS)
        if 'dy' not in state:
            return {'y': y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), state['dy'])
        return {'y': y, 'dx': dx, 'dweight': dw, 'dbias': db}
    if op == 'orth':
        if not own:
            return [t for g in state['groups'] for t in _newton_schulz(g).to(g.dtype).unbind(0)]
        from margipose_amd.train_helpers import orthogonalize
        return orthogonalize(state['matrices'], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    if own:
        state['optimiser'].step()
    else:
        if op == 'muon':
            _plain_muon(state)
        _plain_adamw(state)
    out = {'vectors': state['pv'], 'exp_avg': state['exp_avg'], 'exp_avg_sq': state['exp_avg_sq']}
    if op == 'muon':
        out.update(matrices=state['pm'], momentum=state['momentum'])
    return out


def _exact_orthogonal(g):
    """The same polynomial of one matrix, on the side of its shorter axis, in float64."""
    x = g.double()
    x = x if x.shape[0] >= x.shape[1] else x.t().contiguous()
    x = x / (torch.linalg.vector_norm(x) + NS_EPS)
    eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        h = x.t() @ x
        x = x @ (COEFFICIENTS[0] * eye + h @ (COEFFICIENTS[1] * eye + COEFFICIENTS[2] * h))
    return x if g.shape[0] >= g.shape[1] else x.t().contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'norm':
        x, w = s['x'].detach().double(), s['weight'].detach().double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        xhat = (x - mean) / torch.sqrt(var + LN_EPS)
        out = {'y': xhat * w + s['bias'].detach().double()}
        if 'dy' in s:
            dy = s['dy'].double()
            n = x.shape[1]
            p = dy * w
            out['dbias'] = dy.sum(0)
            out['dweight'] = (dy * xhat).sum(0)
            out['dx'] = (n * p - p.sum(1, keepdim=True) - xhat * (p * xhat).sum(1, keepdim=True)) / (n * torch.sqrt(var + LN_EPS))
        return out
    if case['op'] == 'orth':
        return [_exact_orthogonal(g) for g in s['matrices']]
    gv, pv = _gather(s['gv'], s['texts'][1]).double(), s['pv'].double()
    t = ADAMW_STEPS_BEFORE + 1
    m = ADAMW['momentum'] * s['exp_avg'].double() + (1.0 - ADAMW['momentum']) * gv
    v = ADAMW['beta2'] * s['exp_avg_sq'].double() + (1.0 - ADAMW['beta2']) * gv * gv
    mhat, vhat = m / (1.0 - ADAMW['momentum'] ** t), v / (1.0 - ADAMW['beta2'] ** t)
    out = {'vectors': pv - ADAMW['lr'] * (ADAMW['weight_decay'] * pv + mhat / (torch.sqrt(vhat) + ADAMW['eps'])), 'exp_avg': m, 'exp_avg_sq': v}
    if case['op'] == 'muon':
        gm = _gather(s['gm'], s['texts'][0]).double()
        buf = MUON['momentum'] * s['momentum'].double() + gm
        u = gm + MUON['momentum'] * buf
        p = s['pm'].double()
        p -= MUON['lr'] * MUON['weight_decay'] * p
        for pg, ug in zip(_groups(p, case['shapes']), _groups(u, case['shapes'])):
            for pi, ui in zip(pg, ug):
                pi -= MUON['lr'] * 0.2 * math.sqrt(max(pi.shape)) * _exact_orthogonal(ui)
        out.update(matrices=p, momentum=buf)
    return out


def work(case):
    """Bytes: inputs once, outputs once.  Operations: of the cheaper of two ways to the same polynomial, X on every step or only the
    m x m matrices between X X^T and the last product; a symmetric product is half of one."""
    if case['op'] == 'norm':
        n, size = case['rows'] * case['cols'], torch.empty((), dtype=getattr(torch, case['dtype'])).element_size()
        return {'bytes': n * size * (5 if case['train'] else 2) + 8 * case['cols'] * (2 if case['train'] else 1), 'flops': n * (19 if case['train'] else 8)}
    matrices, vectors = (case['shapes'], case.get('vectors', '')) if case['op'] != 'adamw' else ('', case['shapes'])
    size = {'orth': 2 * torch.empty((), dtype=getattr(torch, case.get('dtype', 'float32'))).element_size(), 'muon': 20, 'adamw': 0}[case['op']]
    nbytes = flops = 0.0
    for k, dims in _shapes(matrices):
        m, n = min(dims), max(dims)
        nbytes += k * size * m * n
        flops += k * min(STEPS * (3.0 * m * m * n + m ** 3), 3.0 * m * m * n + (4 * STEPS - 3) * float(m) ** 3)
    for k, dims in _shapes(vectors):
        nbytes += k * 28.0 * math.prod(dims)
        flops += k * 14.0 * math.prod(dims)
    return {'bytes': nbytes, 'flops': flops}
