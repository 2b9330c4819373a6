"""residual_norm on the GPU against the formulas in 64 bits.

Tolerances.  A stored value is off by half a step of its type, eps / 2 relative (bf16 2^-8, fp16 2^-11, fp32 2^-24), plus the 32-bit arithmetic before
it: every intermediate carries a few roundings of 2^-24 relative to the sum of the magnitudes that enter it.  ``_mags`` carries those sums of
magnitudes through the same formulas (|a| + |b| for a - b), a norm's factor with its condition number mean(|v| + |mean|) / std in front, and a
sum over n terms allows n more roundings of the sum of magnitudes.  64 roundings cover the chain of a row (two norms of at most 13 joining steps each
and the element operations).  fp16 adds half its smallest step, 2^-25."""
import itertools

import pytest
import torch
import torch.utils.checkpoint

from rumpy_amd.residual_norm import ResidualNorm, residual_norm

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U24 = 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


def _stats(v, kind):
    mu = v.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(v[..., :1])
    rs = 1.0 / torch.sqrt(((v - mu) ** 2).mean(-1, keepdim=True) + EPS)
    return mu, rs


def _reference(x, t, gate, group, scale, post, wp, bp, pre, w, b, dy, dh):
    """values and magnitudes in 64 bits -> {name: (value, magnitude, terms)}; rows are 2-D; gate [rows, C] already spread, group = row -> gate row"""
    rows, c = x.shape
    one = torch.ones(c, dtype=torch.float64)
    wpd, wd = one if wp is None else wp, one if w is None else w
    bpd, bd = 0 * one if bp is None else bp, 0 * one if b is None else b
    out = {}
    y, ym = x, x.abs()
    if t is not None:
        g = torch.ones_like(x) if gate is None else gate
        if post:
            mu, rs = _stats(t, post)
            cond = ((t.abs() + mu.abs()) * rs).mean(-1, keepdim=True).clamp(min=1)
            that, thm = (t - mu) * rs, (t.abs() + mu.abs()) * rs * cond
        else:
            rs = torch.ones_like(x[:, :1])
            that, thm = t, t.abs()
        z, zm = that * wpd + bpd, thm * wpd.abs() + bpd.abs()
        y, ym = x + scale * g * z, x.abs() + abs(scale) * g.abs() * zm
        out['y'] = (y, ym, 0)
    if pre:
        mu, rsy = _stats(y, pre)
        cond = ((ym + mu.abs()) * rsy).mean(-1, keepdim=True).clamp(min=1)
        yh, yhm = (y - mu) * rsy, (ym + (ym.mean(-1, keepdim=True) if pre == 'layer' else 0)) * rsy * cond
        out['h'] = (yh * wd + bd, yhm * wd.abs() + bd.abs(), 0)
    d = torch.zeros_like(x) if dy is None else dy
    dm = d.abs()
    if dh is not None:
        a = dh * wd
        am = a.abs()
        s1 = a.mean(-1, keepdim=True) if pre == 'layer' else 0
        s1m = am.mean(-1, keepdim=True) if pre == 'layer' else 0
        d = d + rsy * (a - s1 - yh * (a * yh).mean(-1, keepdim=True))
        dm = dm + rsy * cond * (am + s1m + yhm * (am * yhm).mean(-1, keepdim=True))
        out['d_pre_w'] = ((dh * yh).sum(0), (dh.abs() * yhm).sum(0), rows)
        out['d_pre_b'] = (dh.sum(0), dh.abs().sum(0), rows)
    out['d_x'] = (d, dm, 0)
    if t is not None:
        dz, dzm = scale * g * d, abs(scale) * g.abs() * dm
        dg, dgm = scale * z * d, abs(scale) * zm * dm
        if group is not None:
            n = int(group.max()) + 1
            add = lambda v: torch.zeros(n, c, dtype=torch.float64).index_add_(0, group, v)
            out['d_gate'] = (add(dg), add(dgm), rows)
        elif gate is not None:
            out['d_gate'] = (dg, dgm, 0)
        q, qm = dz * wpd, dzm * wpd.abs()
        if post:
            out['d_post_w'] = ((dz * that).sum(0), (dzm * thm).sum(0), rows)
            out['d_post_b'] = (dz.sum(0), dzm.sum(0), rows)
            s1 = q.mean(-1, keepdim=True) if post == 'layer' else 0
            s1m = qm.mean(-1, keepdim=True) if post == 'layer' else 0
            q, qm = rs * (q - s1 - that * (q * that).mean(-1, keepdim=True)), rs * (qm + s1m + thm * (qm * thm).mean(-1, keepdim=True))
        out['d_branch'] = (q, qm, 0)
    return out


def _check(name, got, ref, dtype):
    value, mag, terms = ref
    got = got.detach().double().cpu().reshape(value.shape)
    tol = STEP[dtype] * value.abs() + (64 + terms) * U24 * mag + (2.0 ** -25 if dtype == F16 else 0.0)
    tol = tol * (1 + STEP[dtype])
    bad = ~((got - value).abs() <= tol)
    assert not bad.any(), '%s: %d of %d off, worst %.3g against %.3g' % (name, int(bad.sum()), bad.numel(), float((got - value).abs()[bad].max()),
                                                                        float(tol[bad].min()))


def _make(shape, tx, tb, gate_kind, post, pre, bias, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    rnd = lambda s, dt=F32, mul=1.0, add=0.0: (torch.randn(s, generator=g) * mul + add).to(dt)
    v = {'x': rnd(shape, tx, 1.5, mean), 'branch': rnd(shape, tb, 0.7, -mean)}
    if gate_kind != 'none':
        gs = {'channel': (c,), 'group': (shape[0], c), 'full': shape}[gate_kind]
        v['gate'] = torch.sigmoid(rnd(gs)).to(tb if gate_kind == 'full' else F32)
    if post:
        v['post_weight'] = rnd((c,), mul=0.2, add=1.0)
        if bias:
            v['post_bias'] = rnd((c,), mul=0.2)
    if pre:
        v['pre_weight'] = rnd((c,), mul=0.2, add=1.0)
        if bias:
            v['pre_bias'] = rnd((c,), mul=0.2)
    return v, rnd(shape, tx), rnd(shape, tb)


def _spread(v, shape, gate_kind):
    """the gate per row, and the gate row of each row"""
    c = shape[-1]
    rows = 1
    for s in shape[:-1]:
        rows *= s
    if gate_kind == 'none':
        return None, None
    g = v['gate'].double()
    if gate_kind == 'full':
        return g.reshape(rows, c), None
    group = torch.zeros(rows, dtype=torch.long) if gate_kind == 'channel' else torch.arange(rows) // (rows // shape[0])
    return g.reshape(-1, c)[group], group


def _run_and_check(shape, tx, tb, gate_kind, post, pre, bias, scale, with_dy=True, with_dh=True, lay=lambda n, t: t, seed=0):
    v, dy, dh = _make(shape, tx, tb, gate_kind, post, pre, bias, seed)
    dev = {n: lay(n, t.to(DEV)).detach().requires_grad_() for n, t in v.items()}
    for n in v:
        assert torch.equal(dev[n].detach().cpu(), v[n])
    y, h = residual_norm(dev['x'], dev['branch'], gate=dev.get('gate'), scale=scale, post_norm=post, post_weight=dev.get('post_weight'),
                         post_bias=dev.get('post_bias'), pre_norm=pre, pre_weight=dev.get('pre_weight'), pre_bias=dev.get('pre_bias'), eps=EPS)
    assert y.dtype == tx and y.shape == torch.Size(shape) and (h is None) == (pre is None)
    outs, grads = [], []
    if with_dy:
        outs.append(y), grads.append(lay('dy', dy.to(DEV)))
    if with_dh and pre:
        outs.append(h), grads.append(lay('dh', dh.to(DEV)))
    got = dict(zip(dev, torch.autograd.grad(outs, list(dev.values()), grads, allow_unused=True)))
    c = shape[-1]
    flat = lambda t: t.double().reshape(-1, c)
    gate, group = _spread(v, shape, gate_kind)
    d64 = lambda n: v[n].double() if n in v else None
    ref = _reference(flat(v['x']), flat(v['branch']), gate, group, scale, post, d64('post_weight'), d64('post_bias'), pre, d64('pre_weight'),
                     d64('pre_bias'), flat(dy) if with_dy else None, flat(dh) if with_dh and pre else None)
    _check('y', y, ref['y'], tx)
    if pre:
        assert h.dtype == tb
        _check('h', h, ref['h'], tb)
    for n, r in (('x', 'd_x'), ('branch', 'd_branch'), ('gate', 'd_gate'), ('post_weight', 'd_post_w'), ('post_bias', 'd_post_b'),
                 ('pre_weight', 'd_pre_w'), ('pre_bias', 'd_pre_b')):
        if n not in v:
            continue
        if r not in ref:
            assert got[n] is None, n
            continue
        assert got[n].dtype == v[n].dtype and got[n].shape == v[n].shape
        _check(r, got[n], ref[r], v[n].dtype)
    return y, h, got


# ---------------------------------------------------------------------------------------------------------------- forward and backward
SHAPES = [(1, 1), (1, 8), (5, 7), (2, 3, 64), (3, 50, 64), (2, 9, 65), (7, 128), (2, 5, 200), (3, 4, 256), (9, 300), (2, 17, 512), (3, 513),
          (2, 3, 1001), (5, 1024), (2, 2, 2047), (3, 2048), (1, 4096), (2, 2, 4097), (3, 8191), (1, 2, 8192), (1, 700, 72), (40, 11, 24)]
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]
FORMS = list(itertools.product((None, 'layer', 'rms'), (None, 'layer', 'rms'), ('none', 'channel', 'group', 'full')))


@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_values_and_gradients_over_shapes(shape):
    """every shape with every pair of types; norms, gates and biases in turn"""
    for i, (tx, tb) in enumerate(TYPES):
        post, pre, gate = FORMS[(7 * i + 5 * SHAPES.index(shape)) % len(FORMS)]
        _run_and_check(shape, tx, tb, gate, post, pre, bias=bool((i + shape[-1]) % 2), scale=(0.1, 1.0, -0.5)[i % 3], seed=i)


@pytest.mark.parametrize('post,pre,gate', FORMS)
def test_values_and_gradients_over_forms(post, pre, gate):
    for shape, (tx, tb) in (((4, 37, 48), (BF16, BF16)), ((2, 3, 1500), (F32, F16))):
        for bias in (False, True):
            _run_and_check(shape, tx, tb, gate, post, pre, bias, 0.3)


@pytest.mark.parametrize('groups,per,c', [(1, 1000, 64), (3, 31, 64), (3, 32, 64), (3, 33, 64), (200, 1, 64), (50, 7, 16), (5, 400, 512), (600, 2, 1024), (7, 3, 8192),
                                          (32, 576, 64)])
def test_gate_rows_of_any_number_of_rows(groups, per, c):
    """a gate row's gradient is summed over its own rows: groups shorter and longer than a workgroup's step, and across workgroups"""
    _run_and_check((groups, per, c), BF16, BF16, 'group', 'layer', 'rms', True, 0.5)


@pytest.mark.parametrize('with_dy,with_dh', [(True, False), (False, True)])
def test_a_gradient_that_does_not_arrive(with_dy, with_dh):
    _run_and_check((3, 20, 96), BF16, BF16, 'group', 'layer', 'layer', True, 0.7, with_dy, with_dh)


def test_norm_in_front_alone():
    for shape, dt, kind in (((5, 64), BF16, 'layer'), ((2, 3, 1001), F32, 'rms'), ((300, 2048), F16, 'layer'), ((7,), F32, 'rms')):
        g = torch.Generator().manual_seed(1)
        x, dh, dy = (torch.randn(shape, generator=g).to(dt) for _ in range(3))
        w, b = torch.randn(shape[-1], generator=g) + 1, torch.randn(shape[-1], generator=g)
        xd, wd, bd = (t.to(DEV).requires_grad_() for t in (x, w, b))
        y, h = residual_norm(xd, pre_norm=kind, pre_weight=wd, pre_bias=bd, eps=EPS)
        assert y is xd
        got = torch.autograd.grad([y, h], [xd, wd, bd], [dy.to(DEV), dh.to(DEV)])
        flat = lambda t: t.double().reshape(-1, shape[-1])
        ref = _reference(flat(x), None, None, None, 1.0, None, None, None, kind, w.double(), b.double(), None, flat(dh))
        _check('h', h, ref['h'], dt)
        # the skip's gradient joins the norm's in torch: one rounding more
        dx = ref['d_x'][0] + flat(dy)
        assert ((got[0].double().cpu().reshape(dx.shape) - dx).abs() <= 2.1 * STEP[dt] * (ref['d_x'][0].abs() + flat(dy).abs()) + 64 * U24 * ref['d_x'][1] + 2.0 ** -24).all()
        _check('d_pre_w', got[1], ref['d_pre_w'], F32)
        _check('d_pre_b', got[2], ref['d_pre_b'], F32)


def test_formulas_are_the_derivatives():
    """the reference's written-out gradients against autograd through the definition, 64 bits, on the CPU"""
    for post, pre, gate_kind in FORMS:
        shape = (2, 3, 5)
        v, dy, dh = _make(shape, F32, F32, gate_kind, post, pre, True)
        leaf = {n: t.double().requires_grad_() for n, t in v.items()}

        def norm(t, kind, w, b):
            if kind is None:
                return t
            mu, rs = _stats(t, kind)
            return (t - mu) * rs * w + b
        g = leaf.get('gate')
        gs = 1.0 if g is None else g[:, None, :] if gate_kind == 'group' else g
        y = leaf['x'] + 0.3 * gs * norm(leaf['branch'], post, leaf.get('post_weight'), leaf.get('post_bias'))
        h = norm(y, pre, leaf.get('pre_weight'), leaf.get('pre_bias'))
        total = (y * dy.double()).sum() + (0 if pre is None else (h * dh.double()).sum())
        got = dict(zip(leaf, torch.autograd.grad(total, list(leaf.values()))))
        gate, group = _spread(v, shape, gate_kind)
        d64 = lambda n: v[n].double() if n in v else None
        flat = lambda t: t.double().reshape(-1, 5)
        ref = _reference(flat(v['x']), flat(v['branch']), gate, group, 0.3, post, d64('post_weight'), d64('post_bias'), pre, d64('pre_weight'), d64('pre_bias'),
                         flat(dy), None if pre is None else flat(dh))
        for n, r in (('x', 'd_x'), ('branch', 'd_branch'), ('gate', 'd_gate'), ('post_weight', 'd_post_w'), ('post_bias', 'd_post_b'),
                     ('pre_weight', 'd_pre_w'), ('pre_bias', 'd_pre_b')):
            if n in v:
                assert torch.allclose(got[n].reshape(ref[r][0].shape), ref[r][0], rtol=1e-10, atol=1e-11), (post, pre, gate_kind, n)


def test_gradient_against_differences():
    """d total / d branch along a direction, central differences of the GPU's own float32 forward pass"""
    v, dy, dh = _make((3, 40, 96), F32, F32, 'group', 'layer', 'rms', True)
    dev = {n: t.to(DEV) for n, t in v.items()}

    def total(moved):
        y, h = residual_norm(moved['x'], moved['branch'], gate=moved['gate'], scale=0.4, post_norm='layer', post_weight=moved['post_weight'],
                             post_bias=moved['post_bias'], pre_norm='rms', pre_weight=moved['pre_weight'], pre_bias=moved['pre_bias'])
        return y, h, (y.double() * dy.to(DEV).double()).sum() + (h.double() * dh.to(DEV).double()).sum()
    for name in v:
        leaf = {n: t.clone().requires_grad_(n == name) for n, t in dev.items()}
        y, h, _ = total(leaf)
        grad, = torch.autograd.grad([y, h], [leaf[name]], [dy.to(DEV), dh.to(DEV)])
        direction = grad / grad.norm()          # along the gradient: the difference is its norm
        step = 1e-2
        up, down = (total({**dev, name: dev[name] + s * step * direction})[2] for s in (1, -1))
        # the step's third-order term and 2^-24-relative noise of about 12 000 summands over 2e-2 both stay below 2e-3 of a norm of order 10
        assert abs(float(up - down) / (2 * step) - float(grad.double().norm())) < 2e-3 * float(grad.norm()) + 1e-2, name


# ---------------------------------------------------------------------------------------------------------------- layouts
def _odd_slice(n, t):
    if t.dim() < 2:
        return t
    wide = torch.zeros(t.shape[:-1] + (t.shape[-1] + 3,), dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def _transposed(n, t):
    return t if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


def _row_gaps(n, t):
    if t.dim() != 3:
        return t
    wide = torch.zeros((t.shape[0], t.shape[1] + 2, t.shape[2]), dtype=t.dtype, device=t.device)
    wide[:, 1:-1] = t
    return wide[:, 1:-1]                      # rows at no common stride


@pytest.mark.parametrize('lay', [_odd_slice, _transposed, _row_gaps], ids=['odd slice', 'transposed', 'row gaps'])
@pytest.mark.parametrize('shape', [(3, 7, 64), (2, 5, 1000)], ids=str)
def test_layouts(lay, shape):
    for tx, tb in TYPES:
        _run_and_check(shape, tx, tb, 'full', 'layer', 'layer', True, 0.5, lay=lay)
        _run_and_check(shape, tx, tb, 'group', 'rms', 'layer', False, 0.5, lay=lay)


def test_expanded_inputs_and_gradients():
    """x one row for all: its gradient comes back summed; upstream gradients of a plain sum are expanded scalars"""
    c = 64
    g = torch.Generator().manual_seed(3)
    row, t = torch.randn(1, c, generator=g), torch.randn(50, c, generator=g)
    rd, td = row.to(DEV).requires_grad_(), t.to(DEV).requires_grad_()
    y, h = residual_norm(rd.expand(50, c), td, post_norm='layer', pre_norm='rms')
    (y.sum() + h.sum()).backward()
    ref = _reference(row.double().expand(50, c), t.double(), None, None, 1.0, 'layer', None, None, 'rms', None, None, torch.ones(50, c).double(), torch.ones(50, c).double())
    _check('row', rd.grad, (ref['d_x'][0].sum(0, keepdim=True), ref['d_x'][1].sum(0, keepdim=True), 50), F32)
    _check('branch', td.grad, ref['d_branch'], F32)


def test_offsets_beyond_32_bits():
    """rows more than 2^31 elements apart"""
    c, stride = 40, 2 ** 31 + 9
    buf = torch.empty(2 * stride + c, dtype=BF16, device=DEV)
    x = buf.as_strided((3, c), (stride, 1))
    g = torch.Generator().manual_seed(4)
    v, t = torch.randn(3, c, generator=g).to(BF16), torch.randn(3, c, generator=g).to(BF16)
    x.copy_(v)
    y, h = residual_norm(x, t.to(DEV), post_norm='rms', pre_norm='layer', eps=EPS)
    ref = _reference(v.double(), t.double(), None, None, 1.0, 'rms', None, None, 'layer', None, None, None, None)
    _check('y', y, ref['y'], BF16)
    _check('h', h, ref['h'], BF16)


# ---------------------------------------------------------------------------------------------------------------- values
def test_not_a_number_stays_in_its_row():
    for bad in (float('nan'), float('inf')):
        v, dy, dh = _make((6, 300), BF16, BF16, 'none', 'layer', 'rms', False)
        v['branch'][2, 7] = bad
        leaf = {n: t.to(DEV).requires_grad_() for n, t in v.items()}
        y, h = residual_norm(leaf['x'], leaf['branch'], post_norm='layer', post_weight=leaf['post_weight'], pre_norm='rms', pre_weight=leaf['pre_weight'])
        dx, dt = torch.autograd.grad([y, h], [leaf['x'], leaf['branch']], [dy.to(DEV), dh.to(DEV)])
        rest = [0, 1, 3, 4, 5]
        for t in (y, h, dx, dt):
            assert torch.isfinite(t[rest]).all() and not torch.isfinite(t[2]).all()


@pytest.mark.parametrize('kind', ['layer', 'rms'])
def test_constant_rows_large_means_and_zeros(kind):
    c = 257
    x = torch.stack([torch.zeros(c), torch.full((c,), 3.0), 1000 + torch.arange(c) % 2.0, torch.full((c,), 1e-20)])
    _, h = residual_norm(x.to(DEV), pre_norm=kind, eps=EPS)
    ref = _reference(x.double(), None, None, None, 1.0, None, None, None, kind, None, None, None, None)
    _check('h', h, ref['h'], F32)


def test_no_rows():
    for shape in ((0, 64), (3, 0, 64), (0, 5, 64)):
        v, _, _ = _make(shape, BF16, BF16, 'group', 'layer', 'layer', True)
        leaf = {n: t.to(DEV).requires_grad_() for n, t in v.items()}
        y, h = residual_norm(leaf['x'], leaf['branch'], gate=leaf['gate'], post_norm='layer', post_weight=leaf['post_weight'], post_bias=leaf['post_bias'],
                             pre_norm='layer', pre_weight=leaf['pre_weight'], pre_bias=leaf['pre_bias'])
        assert y.shape == h.shape == torch.Size(shape)
        grads = torch.autograd.grad([y, h], list(leaf.values()), [torch.zeros_like(y), torch.zeros_like(h)])
        assert all(float(g.abs().sum()) == 0 for g in grads)


# ---------------------------------------------------------------------------------------------------------------- how it is called
def _pass(dev, dy, dh):
    leaf = {n: t.detach().requires_grad_() for n, t in dev.items()}
    y, h = residual_norm(leaf['x'], leaf['branch'], gate=leaf['gate'], scale=0.5, post_norm='layer', post_weight=leaf['post_weight'], post_bias=leaf['post_bias'],
                         pre_norm='rms', pre_weight=leaf['pre_weight'], pre_bias=leaf['pre_bias'])
    return [y.detach(), h.detach()] + list(torch.autograd.grad([y, h], list(leaf.values()), [dy, dh]))


def test_same_bits_every_time_and_on_other_streams():
    v, dy, dh = _make((6, 500, 200), BF16, BF16, 'group', 'layer', 'rms', True)
    dev, dy, dh = {n: t.to(DEV) for n, t in v.items()}, dy.to(DEV), dh.to(DEV)
    first = _pass(dev, dy, dh)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        res = []
        for s in streams:                       # two calls at once
            with torch.cuda.stream(s):
                res.append(_pass(dev, dy, dh))
        torch.cuda.synchronize()
        for r in res:
            assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed():
    """a training pass as one graph, new inputs per replay, eager passes in between"""
    v, dy, dh = _make((4, 100, 96), BF16, BF16, 'group', 'layer', 'rms', True)
    dev, dy, dh = {n: t.to(DEV) for n, t in v.items()}, dy.to(DEV), dh.to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _pass(dev, dy, dh)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(dev, dy, dh)
    g = torch.Generator().manual_seed(9)
    for _ in range(4):
        dev['branch'].copy_(torch.randn(v['branch'].shape, generator=g).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        want = _pass(dev, dy, dh)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_module_is_the_function_and_trains():
    torch.manual_seed(0)
    m = ResidualNorm(96, scale=0.1, post_norm='layer', pre_norm='rms', bias=True, channel_scale=0.5).to(DEV)
    assert {n for n, _ in m.named_parameters()} == {'post_weight', 'post_bias', 'pre_weight', 'pre_bias', 'gate'}
    x, t = torch.randn(4, 10, 96, device=DEV), torch.randn(4, 10, 96, device=DEV)
    y, h = m(x, t)
    y2, h2 = residual_norm(x, t, gate=m.gate, scale=0.1, post_norm='layer', post_weight=m.post_weight, post_bias=m.post_bias, pre_norm='rms',
                           pre_weight=m.pre_weight, pre_bias=m.pre_bias)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    (y.square().mean() + h.square().mean()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    y, h = m(x)
    assert y is x and h.shape == x.shape
    assert {n for n, _ in ResidualNorm(8, pre_norm='rms').named_parameters()} == {'pre_weight'}


def test_backward_twice_of_one_forward():
    v, dy, dh = _make((4, 30, 64), BF16, BF16, 'full', 'layer', 'rms', True)
    leaf = {n: t.to(DEV).requires_grad_() for n, t in v.items()}
    y, h = residual_norm(leaf['x'], leaf['branch'], gate=leaf['gate'], post_norm='layer', post_weight=leaf['post_weight'], post_bias=leaf['post_bias'],
                         pre_norm='rms', pre_weight=leaf['pre_weight'], pre_bias=leaf['pre_bias'])
    grads = [torch.autograd.grad([y, h], list(leaf.values()), [dy.to(DEV), dh.to(DEV)], retain_graph=True) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_no_second_derivative():
    x, t = (torch.randn(3, 64, device=DEV, requires_grad=True) for _ in range(2))
    y, h = residual_norm(x, t, post_norm='rms', pre_norm='rms')
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(y.sum() + h.sum(), [x, t], create_graph=True)


def test_more_than_2_31_elements():
    """rows do not know of each other: those at the end of a large tensor are the rows of a small call, bit for bit"""
    rows, c = 300000, 8192                                        # 2.4e9 elements
    g = torch.Generator(device=DEV).manual_seed(21)
    x, t = (torch.randn((rows, c), generator=g, device=DEV, dtype=BF16) for _ in range(2))
    pick = torch.tensor([0, 1, 131071, 262143, 262144, 299998, 299999], device=DEV)
    res = []
    for some in (None, pick):
        xs, ts = (v if some is None else v[some] for v in (x, t))
        xs, ts = xs.detach().requires_grad_(), ts.detach().requires_grad_()
        y, h = residual_norm(xs, ts, scale=0.3, post_norm='rms', pre_norm='layer')
        dx, dt = torch.autograd.grad([y, h], [xs, ts], [xs.detach(), ts.detach()])
        res.append([v if some is not None else v[pick] for v in (y.detach(), h.detach(), dx, dt)])
        del y, h, dx, dt
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_one_tensor_in_several_places():
    """x as the branch and as its own gate: the gradients of all places come together"""
    g = torch.Generator().manual_seed(22)
    v, dy, dh = (torch.randn(5, 130, generator=g) for _ in range(3))
    d = v.to(DEV).requires_grad_()
    y, h = residual_norm(d, d, gate=d, scale=0.5, post_norm='layer', pre_norm='rms')
    got, = torch.autograd.grad([y, h], d, [dy.to(DEV), dh.to(DEV)])
    ref = _reference(v.double(), v.double(), v.double(), None, 0.5, 'layer', None, None, 'rms', None, None, dy.double(), dh.double())
    _check('y', y, ref['y'], F32)
    parts = [ref[n] for n in ('d_x', 'd_branch', 'd_gate')]
    _check('gradient', got, (sum(p[0] for p in parts), sum(p[1] for p in parts), 3), F32)


def test_modes_around_the_call():
    """inference mode, checkpointing, accumulation into .grad by backward(), a graph that is freed"""
    x, t = torch.randn(6, 72, device=DEV), torch.randn(6, 72, device=DEV)
    w = torch.ones(72, device=DEV, requires_grad=True)
    with torch.inference_mode():
        y0, h0 = residual_norm(x, t, post_norm='rms', post_weight=w, pre_norm='rms')
    y, h = residual_norm(x, t, post_norm='rms', post_weight=w, pre_norm='rms')
    assert torch.equal(y, y0) and torch.equal(h, h0) and not y0.requires_grad and y.requires_grad
    (y.sum() + h.sum()).backward()
    once = w.grad.clone()
    with pytest.raises(RuntimeError, match='second time'):
        y.sum().backward()
    out = torch.utils.checkpoint.checkpoint(lambda a: sum(v.sum() for v in residual_norm(x, t, post_norm='rms', post_weight=a, pre_norm='rms')), w, use_reentrant=False)
    out.backward()
    assert torch.equal(w.grad, 2 * once)
    y, h = residual_norm(x, t, post_norm='rms', post_weight=w, pre_norm='rms')
    t.add_(1.0)                                                   # a saved tensor is changed before the backward pass
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        h.sum().backward()
    with pytest.raises(RuntimeError, match='forward-mode'):
        with torch.autograd.forward_ad.dual_level():
            residual_norm(torch.autograd.forward_ad.make_dual(x, x), t, pre_norm='rms')


def test_captured_backward_accumulates_into_grad():
    """a whole step - forward, loss, backward() into .grad - as one graph, replayed with other inputs and eager steps of other tensors in between"""
    torch.manual_seed(5)
    m = ResidualNorm(64, scale=0.5, post_norm='layer', pre_norm='layer', channel_scale=0.3).to(DEV)
    x, t = torch.randn(40, 64, device=DEV), torch.randn(40, 64, device=DEV)

    def step(m, x, t):
        for p in m.parameters():
            p.grad.zero_()
        y, h = m(x, t)
        (y.square().sum() + (h * x).sum()).backward()
    for p in m.parameters():
        p.grad = torch.zeros_like(p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(m, x, t)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(m, x, t)
    other = ResidualNorm(64, scale=0.5, post_norm='layer', pre_norm='layer', channel_scale=0.3).to(DEV)
    other.load_state_dict(m.state_dict())
    for p in other.parameters():
        p.grad = torch.zeros_like(p)
    for i in range(3):
        t.copy_(torch.randn(40, 64) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        step(other, x, t)
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(m.parameters(), other.parameters()))


@pytest.mark.parametrize('shape', [(1, 64), (37, 5), (301, 72), (1000, 64), (33, 700), (21, 1032), (3, 8192)])
def test_gate_row_for_every_row(shape):
    """a float32 gate beside 16-bit rows: each gate row serves one row, and its gradient is stored, not summed"""
    _run_and_check(shape, BF16, BF16, 'group', 'layer', 'rms', True, 0.7)
    _run_and_check(shape, F32, F16, 'group', None, 'layer', False, 0.7, with_dy=False)


@pytest.mark.parametrize('c', [5, 64, 72, 130, 1000, 4104])
@pytest.mark.parametrize('kind', ['layer', 'rms'])
def test_an_infinity_in_a_row_stays_in_it(kind, c):
    """(v - mean) / sqrt(var + eps) of a row with one infinity: 'rms' has 0 beside NaN, 'layer' NaN alone, at every row length; other rows as without it"""
    g = torch.Generator().manual_seed(c)
    x, t = torch.randn(6, c, generator=g), torch.randn(6, c, generator=g)
    clean = residual_norm(x.to(DEV), t.to(DEV), post_norm=kind, pre_norm=kind)
    alone = residual_norm(x.to(DEV), pre_norm=kind)[1]
    x2, t2 = x.clone(), t.clone()
    x2[1, c - 1] = float('inf')
    t2[4, 0] = -float('inf')
    want = torch.full((c,), float('nan')) if kind == 'layer' else torch.zeros(c)
    keep = torch.tensor([0, 2, 3, 5])
    h = residual_norm(x2.to(DEV), pre_norm=kind)[1]
    last, first = want.clone(), want.clone()
    last[-1] = first[0] = float('nan')
    assert torch.equal(h[1].cpu().isnan(), last.isnan()) and float(h[1].cpu().nan_to_num().abs().max()) == 0.0
    y2, h2 = residual_norm(x.to(DEV), t2.to(DEV), post_norm=kind, pre_norm=kind)
    assert torch.equal(y2[4].cpu().isnan(), first.isnan()) and bool(h2[4].isnan().all())
    if kind == 'rms':
        assert torch.equal(y2[4, 1:].cpu(), x[4, 1:])                     # N_post is 0 there
    for a, b in ((y2, clean[0]), (h2, clean[1])):
        assert torch.equal(a[[0, 1, 2, 3, 5]], b[[0, 1, 2, 3, 5]])
    assert torch.equal(h[keep], alone[keep])


@pytest.mark.parametrize('shape', [(700, 40, 64), (3000, 2, 130), (9000, 3, 5), (513, 4, 40), (40, 3, 8192), (5, 1000, 4100), (300, 33, 513)])
def test_many_gate_rows(shape):
    """gate rows that serve a few rows each, in number: their partial rows lie in one workgroup's part or at the border of two"""
    _run_and_check(shape, BF16, BF16, 'group', 'layer', 'layer', True, 0.7)
    _run_and_check(shape, F32, F32, 'group', None, 'rms', True, -0.4, with_dy=False)


@pytest.mark.parametrize('c', [7, 8, 9, 15, 16, 17, 31, 32, 33])
def test_few_channels(c):
    """one, two, four and eight lanes a row, their rows summed over a wave and over workgroups; groups that end inside a wave's step"""
    for gate, shape in (('none', (1, 1031, c)), ('channel', (3, 700, c)), ('group', (9, 130, c)), ('group', (5, 300, c)), ('full', (1, 517, c))):
        _run_and_check(shape, BF16, BF16, gate, 'layer', 'rms', True, 0.7)
        _run_and_check(shape, F32, F16, gate, 'rms', 'layer', True, 0.7, lay=lambda n, t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2] if t.dim() > 2 else t)


def test_more_elements_of_gate_rows_than_threads():
    """8960000 of them: the threads that sum the gate rows' gradients walk over them"""
    _run_and_check((140000, 2, 64), BF16, BF16, 'group', 'layer', 'layer', True, 0.7)


@pytest.mark.parametrize('shape', [(2, 300, 8192), (8, 260, 2048), (500, 127, 16), (64, 6, 4096), (45, 9, 64), (46, 2, 64), (1, 700, 300)])
def test_gate_rows_on_both_sides_of_their_summing_rule(shape):
    """few long groups of wide rows, many short ones, and numbers beside the border between the two ways of summing a gate row's partial rows"""
    _run_and_check(shape, BF16, BF16, 'group', 'layer', 'layer', True, 0.7)
