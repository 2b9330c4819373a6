"""Work of the residual-norm and distillation operators: cases, inputs, plain forms and the framework's own calls.

Three operators: ``residual_norm`` (y = x + scale * gate * norm(branch), h = norm(y), and the gradients), ``top_logits`` (a teacher's k
largest logits of every row with the log mass of the rest) and ``distill_loss`` (cross-entropy against those top logits, and its
gradient).  ``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, through ``rumpy_amd``."""
import math

import torch

own = False

DEV = 'cuda'
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(name, shape, x, branch, post, pre, gate, bias, scale, train, view=False):
    """shape: "groups,rows of a group,channels"; x / branch: element types of the residual stream and of the block's output;
    gate: 'none', 'channel' [C], 'group' [groups, C] or 'full'; bias: the norms have one; view: the branch is a slice of a wider row"""
    return dict(name=name, op='norm', shape=shape, x=x, branch=branch, post=post, pre=pre, gate=gate, bias=bias, scale=scale, train=train, view=view)


def _top(name, rows, cols, k, dtype, tau, view=False):
    return dict(name=name, op='top', rows=rows, cols=cols, k=k, dtype=dtype, tau=tau, view=view)


def _distill(name, rows, cols, k, dtype, tau, rest, padded, train, view=False):
    """rest: the teacher's mass outside its top logits is one more outcome; padded: the last rows of every 64 carry weight 0"""
    return dict(name=name, op='distill', rows=rows, cols=cols, k=k, dtype=dtype, tau=tau, rest=rest, padded=padded, train=train, view=view)


def listed():
    return [
        # one token of a deep residual network being served: latency alone
        _norm('norm_one_token', '1,1,4096', 'bf16', 'bf16', 'rms', 'rms', 'none', False, 0.1, False),
        # evaluation of 64-feature activations, a batch of 32 crops of 48 x 48, one channel gate per image
        _norm('norm_pixels_eval', '32,2304,64', 'bf16', 'bf16', 'layer', 'layer', 'group', True, 1.0, False),
        # the training step over the same activations
        _norm('norm_pixels_train', '32,2304,64', 'bf16', 'bf16', 'layer', 'layer', 'group', True, 0.1, True),
        # a training step over tokens, a gate for each element, as a gated block makes it
        _norm('norm_tokens_train', '1,8192,4096', 'bf16', 'bf16', 'rms', 'rms', 'full', False, 1.0, True),
        # a residual stream kept in 32 bits with blocks in 16, odd sizes, a learnt scale for each channel, the branch a slice of a wider row
        _norm('norm_odd_train', '3,1367,1001', 'f32', 'bf16', 'layer', 'layer', 'channel', True, 1.0, True, view=True),
        # the momentum teacher's similarities to the queue of 8192 keys, behind the column of the positive key
        _top('top_queue', 32, 8192, 64, 'f32', 0.07, view=True),
        # a teacher's logits over a large vocabulary of odd size
        _top('top_vocabulary', 2048, 65521, 100, 'bf16', 1.0),
        # few rows, very long
        _top('top_long_rows', 3, 262144, 256, 'f16', 2.0),
        # the contrastive step's loss: 32 queries against the queue
        _distill('distill_queue_train', 32, 8192, 64, 'f32', 0.2, True, False, True, view=True),
        # a training batch of sequences with padding, odd vocabulary
        _distill('distill_vocabulary_train', 4096, 50021, 64, 'bf16', 1.0, True, True, True),
        # scoring a batch without a gradient, renormalised top logits
        _distill('distill_score', 1000, 32000, 16, 'f32', 4.0, False, False, False),
        # few rows, very long
        _distill('distill_long_rows_train', 2, 262144, 256, 'f16', 2.0, False, False, True),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'top', 'distill', 'distill'])
    if op == 'norm':
        c = _logint(rng, 8, 8192)
        rows = _logint(rng, 1, min(131072, 8192 * 4096 // c))
        groups = rng.choice([1, rng.randint(1, 64)])
        per = max(1, rows // groups)
        x, b = rng.choice([('bf16', 'bf16'), ('f32', 'bf16'), ('f32', 'f32'), ('f16', 'f16'), ('f32', 'f16')])
        case = _norm('', '%d,%d,%d' % (groups, per, c), x, b, rng.choice(['layer', 'rms', 'none']), rng.choice(['layer', 'rms']),
                     rng.choice(['none', 'channel', 'group', 'full']), rng.random() < 0.5, rng.choice([0.1, 0.5, 1.0]), rng.random() < 0.6,
                     view=rng.random() < 0.3)
    elif op == 'top':
        cols = _logint(rng, 512, 262144)
        rows = _logint(rng, 1, min(16384, 2048 * 65521 // cols))
        case = _top('', rows, cols, _logint(rng, 1, 256), rng.choice(['f32', 'bf16', 'f16']), rng.choice([0.07, 0.5, 1.0, 2.0]), view=rng.random() < 0.3)
    else:
        cols = _logint(rng, 512, 262144)
        rows = _logint(rng, 1, min(16384, 2048 * 65521 // cols))
        case = _distill('', rows, cols, _logint(rng, 1, 256), rng.choice(['f32', 'bf16', 'f16']), rng.choice([0.2, 1.0, 2.0, 4.0]), rng.random() < 0.5,
                        rng.random() < 0.5, rng.random() < 0.6, view=rng.random() < 0.3)
    del case['name']
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype=torch.float32, mul=1.0, add=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * mul + add).to(dtype)


def _sliced(g, shape, dtype, mul):
    """the last channels of rows that are one element wider: odd row stride, odd alignment"""
    wide = _randn(g, tuple(shape[:-1]) + (shape[-1] + 1,), dtype, mul)
    return wide[..., 1:]


def prepare(case, seed):
    g = _gen(seed)
    st = {'case': case}
    if case['op'] == 'norm':
        n, r, c = (int(v) for v in case['shape'].split(','))
        tx, tb = DTYPES[case['x']], DTYPES[case['branch']]
        make = _sliced if case['view'] else _randn
        st['x'] = _randn(g, (n, r, c), tx, 1.5)
        st['branch'] = make(g, (n, r, c), tb, 0.7)
        st['gate'] = {'none': None, 'channel': (c,), 'group': (n, c), 'full': (n, r, c)}[case['gate']]
        if st['gate'] is not None:          # gates lie between 0 and 1
            st['gate'] = torch.sigmoid(_randn(g, st['gate'])).to(tb if case['gate'] == 'full' else torch.float32)
        for which in ('post', 'pre'):
            normed = case[which] != 'none'
            st[which + '_weight'] = _randn(g, (c,), mul=0.2, add=1.0) if normed else None
            st[which + '_bias'] = _randn(g, (c,), mul=0.2) if normed and case['bias'] else None
        if case['train']:
            st['dy'] = _randn(g, (n, r, c), tx, 0.01)
            st['dh'] = _randn(g, (n, r, c), tb, 0.01)
        return st
    rows, cols, k, dt = case['rows'], case['cols'], case['k'], DTYPES[case['dtype']]
    spread = 3.0 * min(1.0, case['tau'])
    if case['op'] == 'top':
        st['logits'] = (_sliced if case['view'] else _randn)(g, (rows, cols), dt, spread)
        return st
    student = _randn(g, (rows, cols + 1 if case['view'] else cols), dt, spread)
    st['logits'] = student[:, 1:] if case['view'] else student
    teacher = st['logits'].float()
    teacher = teacher + _randn(g, teacher.shape, mul=0.5 * spread)
    st['top_values'], st['top_indices'] = torch.topk(teacher, k, dim=1)
    st['tail'] = torch.logsumexp((teacher / case['tau']).scatter(1, st['top_indices'], -math.inf), dim=1) if case['rest'] else None
    st['top_values'] = st['top_values'].to(dt)
    st['row_weight'] = ((torch.arange(rows, device=DEV) % 64) < 50).float() if case['padded'] else None
    # 16-bit floats with 5 exponent bits train with a loss scale: the gradient of a mean over many rows would vanish in them
    st['upstream'] = torch.tensor(64.0 * rows if case['dtype'] == 'f16' else 1.0, device=DEV)
    return st


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(v, kind, weight, bias, eps):
    if kind == 'none':
        return v
    if kind == 'layer':
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def _leaves(st, names):
    return {n: st[n].detach().requires_grad_() for n in names if st.get(n) is not None}


NORM_LEAVES = ('x', 'branch', 'gate', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')
EPS = 1e-5


def _forward_norm(case, v):
    if own:
        from rumpy_amd.residual_norm import residual_norm
        return residual_norm(v['x'], v['branch'], gate=v.get('gate'), scale=case['scale'], post_norm=None if case['post'] == 'none' else case['post'],
                             post_weight=v.get('post_weight'), post_bias=v.get('post_bias'), pre_norm=case['pre'], pre_weight=v.get('pre_weight'),
                             pre_bias=v.get('pre_bias'), eps=EPS)
    z = _plain_norm(v['branch'].float(), case['post'], v.get('post_weight'), v.get('post_bias'), EPS)
    gate = v.get('gate')
    if gate is not None:
        z = z * (gate.float().unsqueeze(1) if case['gate'] == 'group' else gate.float())
    y = v['x'].float() + case['scale'] * z
    h = _plain_norm(y, case['pre'], v.get('pre_weight'), v.get('pre_bias'), EPS)
    return y.to(v['x'].dtype), h.to(v['branch'].dtype)


def _run_norm(st):
    case = st['case']
    if not case['train']:
        with torch.no_grad():
            y, h = _forward_norm(case, st)
        return {'y': y, 'h': h}
    v = _leaves(st, NORM_LEAVES)
    y, h = _forward_norm(case, v)
    grads = torch.autograd.grad((y, h), list(v.values()), (st['dy'], st['dh']))
    out = {'y': y.detach(), 'h': h.detach()}
    out.update(('d_' + n, gr) for n, gr in zip(v, grads))
    return out


def _plain_lse(u):
    m = u.amax(-1, keepdim=True)
    return (m + torch.log(torch.exp(u - m).sum(-1, keepdim=True))).squeeze(-1)


def _run_top(st):
    case, logits = st['case'], st['logits']
    if own:
        from rumpy_amd.distill import top_logits
        values, indices, tail = top_logits(logits, case['k'], temperature=case['tau'])
        return {'values': values, 'indices': indices, 'tail': tail}
    cols = logits.shape[1]
    # one sortable integer for (value, index), so that equal values go to the lowest index
    bits = (logits.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    key = order * 2 ** 31 + (cols - 1 - torch.arange(cols, device=logits.device))
    indices = cols - 1 - torch.topk(key, case['k'], dim=1)[0] % 2 ** 31
    tail = _plain_lse((logits.float() / case['tau']).scatter(1, indices, -math.inf))
    return {'values': torch.gather(logits, 1, indices), 'indices': indices, 'tail': tail}


def _plain_distill(z, st):
    tau, idx = st['case']['tau'], st['top_indices']
    u = z.float() / tau
    lse = _plain_lse(u)
    v = st['top_values'].float() / tau
    listed_q = torch.gather(u, 1, idx) - lse.unsqueeze(1)
    if st['tail'] is None:
        logp = v - _plain_lse(v).unsqueeze(1)
        rows = (torch.exp(logp) * (logp - listed_q)).sum(1)
    else:
        total = _plain_lse(torch.cat([v, st['tail'].unsqueeze(1)], 1))
        logp, logp_rest = v - total.unsqueeze(1), st['tail'] - total
        logq_rest = _plain_lse(u.scatter(1, idx, -math.inf)) - lse
        rows = (torch.exp(logp) * (logp - listed_q)).sum(1) + torch.exp(logp_rest) * (logp_rest - logq_rest)
    rows = rows * tau ** 2
    w = st['row_weight']
    return rows.mean() if w is None else (rows * w).sum() / w.sum()


def _run_distill(st):
    case = st['case']
    z = st['logits'].detach()
    if case['train']:
        z.requires_grad_()
    if own:
        from rumpy_amd.distill import distill_loss
        loss = distill_loss(z, st['top_values'], st['top_indices'], tail=st['tail'], temperature=case['tau'], row_weight=st['row_weight'])
    else:
        loss = _plain_distill(z, st)
    if not case['train']:
        return {'loss': loss}
    return {'loss': loss.detach(), 'd_logits': torch.autograd.grad(loss, z, st['upstream'])[0]}


def run(state):
    return {'norm': _run_norm, 'top': _run_top, 'distill': _run_distill}[state['case']['op']](state)


# ---------------------------------------------------------------------------------------------------------------- bytes and operations
def work(case):
    if case['op'] == 'norm':
        n, r, c = (int(v) for v in case['shape'].split(','))
        e, bx, bb = n * r * c, BYTES[case['x']], BYTES[case['branch']]
        gate = {'none': 0, 'channel': 4 * c, 'group': 4 * n * c, 'full': bb * e}[case['gate']]
        params = 4 * c * ((case['post'] != 'none') + (case['pre'] != 'none')) * (2 if case['bias'] else 1)
        total = e * 2 * (bx + bb) + gate + params                    # x, branch, y, h
        flops = 16 * e
        if case['train']:
            total += e * 2 * (bx + bb) + gate + params               # dy, dh, dx, d branch
            flops += 34 * e
        return {'bytes': total, 'flops': flops}
    rows, cols, k, b = case['rows'], case['cols'], case['k'], BYTES[case['dtype']]
    if case['op'] == 'top':
        return {'bytes': rows * (cols * b + k * (b + 8) + 4), 'flops': 4 * rows * cols}
    total, flops = rows * (cols * b + k * (b + 8) + (4 if case['rest'] else 0) + (4 if case['padded'] else 0)), 4 * rows * cols
    if case['train']:
        total, flops = total + rows * cols * b, flops + 4 * rows * cols
    return {'bytes': total, 'flops': flops}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_norm(case, st):
    """the formulas with the gradients written out, in 64 bits"""
    d = lambda name: None if st.get(name) is None else st[name].double()
    x, t, gate = d('x'), d('branch'), d('gate')
    gate_b = torch.ones_like(t) if gate is None else (gate[:, None, :] if case['gate'] == 'group' else gate).expand_as(t)

    def stats(v, kind):
        mu = v.sum(-1, keepdim=True) / v.shape[-1] if kind == 'layer' else torch.zeros_like(v[..., :1])
        return mu, 1.0 / torch.sqrt(((v - mu) ** 2).sum(-1, keepdim=True) / v.shape[-1] + EPS)

    def affine(hat, which):
        out = hat * d(which + '_weight')
        return out if st[which + '_bias'] is None else out + d(which + '_bias')

    def back(grad_hat, hat, rs, kind):
        out = grad_hat - hat * (grad_hat * hat).sum(-1, keepdim=True) / hat.shape[-1]
        if kind == 'layer':
            out = out - grad_hat.sum(-1, keepdim=True) / hat.shape[-1]
        return out * rs

    if case['post'] != 'none':
        mu_t, rs_t = stats(t, case['post'])
        t_hat = (t - mu_t) * rs_t
        z = affine(t_hat, 'post')
    else:
        z = t
    y = x + case['scale'] * gate_b * z
    mu_y, rs_y = stats(y, case['pre'])
    y_hat = (y - mu_y) * rs_y
    out = {'y': y, 'h': affine(y_hat, 'pre')}
    if not case['train']:
        return out
    dy, dh = d('dy'), d('dh')
    rows = lambda v: v.reshape(-1, v.shape[-1]).sum(0)
    full = dy + back(dh * d('pre_weight'), y_hat, rs_y, case['pre'])
    dz = case['scale'] * gate_b * full
    out['d_x'] = full
    out['d_branch'] = back(dz * d('post_weight'), t_hat, rs_t, case['post']) if case['post'] != 'none' else dz
    if gate is not None:
        dg = case['scale'] * z * full
        out['d_gate'] = {'channel': rows, 'group': lambda v: v.sum(1), 'full': lambda v: v}[case['gate']](dg)
    if case['post'] != 'none':
        out['d_post_weight'] = rows(dz * t_hat)
        if st['post_bias'] is not None:
            out['d_post_bias'] = rows(dz)
    out['d_pre_weight'] = rows(dh * y_hat)
    if st['pre_bias'] is not None:
        out['d_pre_bias'] = rows(dh)
    return out


def _exact_top(case, st):
    """a stable sort of every row, largest first"""
    logits = st['logits']
    values, order = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    k = case['k']
    rest = values[:, k:] / case['tau']
    top = rest[:, :1]
    tail = top[:, 0] + torch.log(torch.exp(rest - top).sum(1))
    return {'values': values[:, :k], 'indices': order[:, :k], 'tail': tail}


def _exact_distill(case, st):
    """probabilities and the gradient written out, in 64 bits"""
    tau, idx = case['tau'], st['top_indices']
    u = st['logits'].double() / tau
    q = torch.exp(u - u.max(1, keepdim=True)[0])
    q = q / q.sum(1, keepdim=True)
    v = st['top_values'].double() / tau
    listed_mask = torch.zeros(u.shape, dtype=torch.bool, device=u.device).scatter_(1, idx, True)
    q_listed = torch.gather(q, 1, idx)
    if st['tail'] is None:
        p = torch.exp(v - v.max(1, keepdim=True)[0])
        p = p / p.sum(1, keepdim=True)
        rows = (p * torch.log(p / q_listed)).sum(1)
        off = q
    else:
        rest = st['tail'].double()[:, None]
        m = torch.maximum(v.max(1, keepdim=True)[0], rest)
        p, p_rest = torch.exp(v - m), torch.exp(rest - m)
        total = p.sum(1, keepdim=True) + p_rest
        p, p_rest = p / total, p_rest / total
        q_rest = (q * ~listed_mask).sum(1, keepdim=True)
        rows = (p * torch.log(p / q_listed)).sum(1) + (p_rest * torch.log(p_rest / q_rest))[:, 0]
        off = q * (1.0 - p_rest / q_rest)
    w = torch.ones(u.shape[0], dtype=torch.float64, device=u.device) if st['row_weight'] is None else st['row_weight'].double()
    w = w / w.sum()
    out = {'loss': tau * tau * (w * rows).sum()}
    if case['train']:
        out['d_logits'] = torch.where(listed_mask, q - torch.zeros_like(q).scatter_(1, idx, p), off) * (tau * w * st['upstream'].double())[:, None]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {'norm': _exact_norm, 'top': _exact_top, 'distill': _exact_distill}[case['op']](case, st)
