"""top_logits and distill_loss on the GPU against their definitions in 64 bits.

Tolerances.  With u = z / T, the exponent of a column is off by a few roundings (2^-24) of |u - max u| (the product with log2(e) / T, both
rounded, and the exponential's own last bits), and a row's sum by as many roundings as it has joining steps, at most V / 4096 pieces of 8 per thread and
13 more: E = 2^-24 (8 max|u - max u| + 64 + V / 256) relative for a probability, absolute for a logarithm.  A stored gradient adds half a step of its
type (bf16 2^-8, fp16 2^-11 and at least 2^-25, fp32 2^-24, relative).  The exponential gives 0 where its result lies under the smallest normal
number: a column's q and p may each be off by 2^-126 for that, its gradient by 2 x 2^-126 times the row's factor (T, weight, upstream)."""
import math

import pytest
import torch

from rumpy_amd.distill import distill_loss, top_logits
from rumpy_amd.sr_tools.loss_functions import TopLogitsDistillLoss

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U24 = 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LOWEST = {t: torch.finfo(t).min for t in STEP}
INF, NAN = math.inf, math.nan


# ---------------------------------------------------------------------------------------------------------------- top_logits
def _top_reference(z, k, tau):
    values, order = torch.sort(z.double() + 0.0, dim=-1, descending=True, stable=True)         # NaN first, equal values by index
    rest = values[..., k:] / tau
    tail = torch.logsumexp(rest, -1) if rest.shape[-1] else torch.full(z.shape[:-1], -INF, dtype=torch.float64)
    return order[..., :k], tail


def _check_top(z, k, tau):
    values, indices, tail = top_logits(z, k, temperature=tau)
    zc = z.cpu()
    order, want = _top_reference(zc, k, tau)
    assert indices.dtype == torch.int64 and values.dtype == z.dtype and tail.dtype == F32
    assert torch.equal(indices.cpu(), order)
    got = torch.gather(zc, -1, order)
    assert torch.equal(values.cpu().nan_to_num(7.0, 8.0, 9.0), got.nan_to_num(7.0, 8.0, 9.0))
    tail = tail.double().cpu()
    # (float32 holds it: a type's lowest value over a temperature under 1, -3.4e38 / 0.5, lies beyond the largest number 2^128 (1 - 2^-24) and rounds to -inf)
    want = want.masked_fill(want < -(2.0 ** 128) * (1 - 2.0 ** -25), -INF)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(tail), torch.isnan(want)) and torch.equal(tail[~finite].nan_to_num(1.0), want[~finite].nan_to_num(1.0))
    if finite.any():
        u = torch.where(torch.isfinite(zc.double()), zc.double() / tau, torch.zeros((), dtype=torch.float64))
        mag = u.abs().amax(-1)
        tol = U24 * (8 * mag + 64 + zc.shape[-1] / 256) + U24 * want.abs()
        assert ((tail - want).abs() <= tol)[finite].all(), float(((tail - want).abs() / tol)[finite].max())


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rows,cols,ks', [(3, 1, (1,)), (2, 2, (1, 2)), (5, 63, (1, 63)), (4, 300, (5, 256)), (3, 512, (1, 256)), (3, 513, (1, 7, 256)), (5, 1000, (64, 256)),
                                          (3, 4095, (100,)), (3, 4096, (100, 256)), (2, 8192, (64,)), (33, 8193, (64,)), (2, 50021, (1, 256)),
                                          (1, 262144, (17, 256)), (700, 600, (8,))])
def test_top_logits_over_sizes(rows, cols, ks, dtype):
    g = torch.Generator().manual_seed(rows * cols)
    z = torch.randn(rows, cols, generator=g).mul(3).to(dtype).to(DEV)
    for k in ks:
        for tau in (1.0, 0.07, 4.0):
            _check_top(z, k, tau)


@pytest.mark.parametrize('cols', [200, 900, 5000, 70001])
def test_top_logits_with_equal_values(cols):
    """rows that are constant, of few distinct values, ascending, descending; zeros of both signs"""
    j = torch.arange(cols, dtype=F32)
    g = torch.Generator().manual_seed(cols)
    z = torch.stack([torch.full((cols,), 2.5), j % 3, j / cols, -j / cols, torch.where(j % 2 == 0, 0.0, -0.0),
                     torch.randint(0, 40, (cols,), generator=g).float(), (j >= cols - 70).float(), (j < 70).float()])
    for dtype in (F32, BF16):
        for k in (1, 64, 200):
            _check_top(z.to(dtype).to(DEV), k, 1.0)


@pytest.mark.parametrize('cols', [300, 3000, 20000])
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
def test_top_logits_with_masks_and_odd_values(cols, dtype):
    g = torch.Generator().manual_seed(cols)
    base = torch.randn(12, cols, generator=g)
    z = base.clone()
    z[0, 50:] = -INF                        # fewer finite values than k
    z[1, 100:] = LOWEST[dtype]
    z[2] = -INF                             # nothing at all
    z[3] = LOWEST[dtype]
    z[4, 17] = NAN
    z[5, [3, 250]] = INF
    z[6, torch.randperm(cols, generator=g)[:280]] = INF       # more than k
    z[7, ::2] = -INF
    z[8, torch.randperm(cols, generator=g)[:290]] = NAN
    z[9, 64:] = -INF                        # exactly k
    z[10, 64:] -= 300.0                     # a gap that no 32-bit exponential spans
    z[11, 100:] -= 300.0
    z = z.to(dtype).to(DEV)
    for tau in (1.0, 4.0):
        _check_top(z, 64, tau)


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rows,cols,offset', [(1, 32768, 0), (3, 32769, 1), (2, 65537, 3), (5, 100000, 5), (1, 270001, 7), (1, 73729, 0), (130, 33001, 1)])
def test_top_logits_of_rows_that_are_cut(rows, cols, offset, dtype):
    """few long rows: the pieces' own selections and their join, with pieces that hold everything, nothing, equal values or a short end"""
    g = torch.Generator().manual_seed(cols)
    z = torch.zeros(rows, cols + 8)
    z[:, offset:offset + cols] = torch.randn(rows, cols, generator=g).mul(3)
    z[0, offset:offset + 9000] += 20.0               # the first piece has all of the top
    if rows > 1:
        z[1] = (torch.arange(cols + 8) % 5).float()
    if rows > 2:
        z[2, 100:] = -INF
        z[2, offset + cols - 30:] = 1.0
    for i in range(3, min(rows, 6)):
        z[i, offset + 17 * i] = (NAN, INF, -INF)[i - 3]
    z = z.to(dtype).to(DEV)[:, offset:offset + cols]
    for k in (1, 100, 256):
        _check_top(z, k, 0.5)


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rows,cols', [(3, 9000), (1100, 3000), (2, 70000)])
def test_top_logits_where_masks_leave_a_few_columns(rows, cols, dtype):
    """a run of valid columns at the front, in the middle, at the end, or every so many: enough for k in some waves' share, in few threads, or hardly"""
    g = torch.Generator().manual_seed(cols)
    base = torch.randn(rows, cols, generator=g)
    for mask in (-INF, LOWEST[dtype]):
        for lo, hi, step in ((0, 2000, 1), (cols // 2, cols // 2 + 700, 1), (cols - 90, cols, 1), (5, cols, 40), (0, 64, 1)):
            z = torch.full((rows, cols), mask)
            z[:, lo:hi:step] = base[:, lo:hi:step]
            _check_top(z.to(dtype).to(DEV), 64, 1.0)


def test_top_logits_of_slices_and_leading_dimensions():
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(6, 8200, generator=g).to(DEV)
    _check_top(wide[:, 1:], 64, 0.07)
    _check_top(wide[:, 3:8003].to(BF16)[:, 5:], 10, 1.0)
    _check_top(torch.randn(2, 3, 4, 700, generator=g).to(DEV), 9, 1.0)
    _check_top(torch.randn(900, 4, generator=g).to(DEV).t(), 9, 1.0)
    _check_top(torch.randn(1, 700, generator=g).to(DEV).expand(5, 700), 9, 1.0)
    _check_top(torch.randn(700, generator=g).to(DEV), 9, 1.0)
    for shape in ((0, 700), (3, 0, 700)):
        values, indices, tail = top_logits(torch.zeros(shape, device=DEV), 5)
        assert values.shape == indices.shape == torch.Size(shape[:-1] + (5,)) and tail.shape == torch.Size(shape[:-1])


def test_offsets_beyond_32_bits():
    cols, stride = 3000, 2 ** 31 + 9
    buf = torch.empty(2 * stride + cols, dtype=BF16, device=DEV)
    z = buf.as_strided((3, cols), (stride, 1))
    g = torch.Generator().manual_seed(4)
    z.copy_(torch.randn(3, cols, generator=g).to(BF16))
    _check_top(z, 20, 1.0)
    values, indices, tail = top_logits(z, 20)
    # (the order of a row's sum goes with the alignment of its address: not the same bits as for a copy of the rows)
    got = distill_loss(z, values, indices, tail=tail, reduction='none').double().cpu()
    one = torch.ones(3, dtype=torch.float64)
    loss, _, _, err, _ = _loss_reference(z.cpu(), values.cpu(), indices.cpu(), tail.cpu(), 1.0, one, one)
    assert ((got - loss).abs() <= 3 * err).all()


# ---------------------------------------------------------------------------------------------------------------- distill_loss
def _loss_reference(z, values, indices, tail, tau, weight, upstream):
    """64 bits: weighted row losses, d (upstream . row losses) / d z, and the relative error E of a probability of each row"""
    rows, cols = z.shape
    u = z.double() / tau
    used = indices >= 0
    idx = indices.clamp(min=0).long()
    v = torch.where(used, values.double() / tau, torch.full((), -INF, dtype=torch.float64))
    listed = torch.zeros(rows, cols, dtype=torch.bool)
    for r in range(rows):
        listed[r, idx[r][used[r]]] = True
    lse = torch.logsumexp(u, 1, keepdim=True)
    lq = u - lse
    parts = v if tail is None else torch.cat([v, tail.double()[:, None]], 1)
    total = torch.logsumexp(parts, 1, keepdim=True)
    says = total[:, 0] > -INF
    lp = parts - torch.where(says[:, None], total, torch.zeros((), dtype=torch.float64))
    p = torch.exp(lp)
    lqs = torch.gather(lq, 1, idx)
    if tail is not None:
        rest = torch.where(listed, torch.full((), -INF, dtype=torch.float64), u)
        lrest = torch.logsumexp(rest, 1, keepdim=True)
        lqs = torch.cat([lqs, lrest - lse], 1)
    terms = torch.where(p > 0, p * (lp - lqs), torch.zeros((), dtype=torch.float64))
    loss = tau ** 2 * terms.sum(1)
    q = torch.exp(lq)
    share = torch.zeros(rows, cols, dtype=torch.float64).scatter_add_(1, idx, torch.where(used, p[:, :idx.shape[1]], torch.zeros((), dtype=torch.float64)))
    grad = q - share
    mag = q + share
    if tail is not None:
        r = torch.exp(rest - lrest)
        pt = p[:, -1:]
        qt = torch.exp(lrest - lse)
        r = torch.where(torch.isfinite(lrest), r, torch.zeros_like(r))
        grad = torch.where(listed, grad, r * (qt - pt))
        mag = torch.where(listed, mag, r * (qt + pt))
    live = says & (weight != 0)
    loss = torch.where(live, loss * weight, torch.zeros_like(loss))
    scale = torch.where(live, tau * weight * upstream, torch.zeros_like(loss))[:, None]
    grad = torch.where(live[:, None], grad * scale, torch.zeros_like(grad))
    mag = torch.where(live[:, None], mag * scale.abs(), torch.zeros_like(mag))
    fin = torch.isfinite(u)
    span = torch.where(fin, u, torch.full((), -INF, dtype=torch.float64)).amax(1) - torch.where(fin, u, torch.full((), INF, dtype=torch.float64)).amin(1)
    vfin = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    span = torch.nan_to_num(span, 0.0, 0.0, 0.0).clamp(min=0) + (vfin.amax(1) - vfin.amin(1)) + (0 if tail is None else torch.nan_to_num(tail.double(), 0, 0, 0).abs() + vfin.abs().amax(1))
    return loss, grad, mag, U24 * (8 * span + 64 + cols / 256), 2 * 2.0 ** -126 * scale.abs()


def _teacher(z, k, tau, rest, g):
    t = (z.double() + 0.5 * torch.randn(z.shape, generator=g)).float()
    v, i = torch.sort(t, dim=1, descending=True, stable=True)
    tail = torch.logsumexp(v[:, k:].double() / tau, 1).float() if rest else None
    return v[:, :k].contiguous(), i[:, :k].contiguous(), tail


def _check_loss(z, values, indices, tail, tau, weight=None, lay=lambda t: t):
    """all three reductions, each with its gradient; z on the CPU"""
    rows = z.shape[0]
    w = torch.ones(rows, dtype=torch.float64) if weight is None else weight.double()
    dev = lambda t: None if t is None else t.to(DEV)
    for reduction in ('none', 'sum', 'mean'):
        zd = lay(z.to(DEV)).detach().requires_grad_()
        got = distill_loss(zd, dev(values), dev(indices), tail=dev(tail), temperature=tau, row_weight=dev(weight), reduction=reduction)
        f = 1.0 if reduction != 'mean' else (1.0 / float(w.sum()) if float(w.sum()) else 0.0)
        # a loss scale, as 16-bit floats of 5 exponent bits need it
        up = torch.linspace(0.5, 2.0, rows).mul(32) if reduction == 'none' else torch.tensor(64.0 * rows)
        grad, = torch.autograd.grad(got, zd, up.to(DEV))
        loss, want, mag, err, tiny = _loss_reference(z, values, indices, tail, tau, w, up.float().double() * f)
        tol_rows = tau ** 2 * w.abs() * 3 * err + 16 * U24 * loss.abs()
        finite = torch.isfinite(loss)
        if reduction == 'none':
            assert got.shape == torch.Size([rows])
            res = got.detach().double().cpu()
            assert torch.equal(torch.isnan(res), torch.isnan(loss)) and torch.equal(res[~finite].nan_to_num(1.0), loss[~finite].nan_to_num(1.0))
            assert ((res - loss).abs() <= tol_rows)[finite].all()
        elif finite.all():
            tol = f * float(tol_rows.sum() + rows * U24 * loss.abs().sum())
            assert abs(float(got.detach()) - f * float(loss.sum())) <= tol, (float(got), f * float(loss.sum()), tol)
        assert grad.dtype == z.dtype and grad.shape == z.shape
        grad = grad.double().cpu()
        step = STEP[z.dtype]
        tol = (step * want.abs() + 3 * err[:, None] * mag) * (1 + step) + (2.0 ** -25 if z.dtype == F16 else 2.0 ** -126) + tiny
        assert torch.equal(torch.isnan(grad), torch.isnan(want))
        ok = torch.isnan(want) | ((grad - want).abs() <= tol)
        assert bool(ok.all()), (reduction, int((~ok).sum()), float(((grad - want).abs() / tol)[~ok].max()))


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('rows,cols,k', [(1, 1, 1), (3, 2, 1), (4, 7, 7), (5, 100, 64), (3, 256, 256), (6, 4095, 17), (4, 4097, 1), (8, 8192, 64), (3, 8193, 256),
                                         (2, 40001, 100), (1, 300000, 256), (70, 1000, 5)])
def test_loss_and_gradient_over_sizes(rows, cols, k, rest, dtype):
    g = torch.Generator().manual_seed(rows + cols + k)
    z = torch.randn(rows, cols, generator=g).mul(3).to(dtype)
    for tau in (1.0, 0.2, 4.0):
        values, indices, tail = _teacher(z, k, tau, rest, g)
        _check_loss(z, values.to(dtype), indices if tau == 1.0 else indices.int(), tail, tau)


@pytest.mark.parametrize('rest', [False, True])
def test_padded_rows_are_not_looked_at(rest):
    g = torch.Generator().manual_seed(2)
    for cols in (900, 20000):               # whole rows, and rows that are cut
        z = torch.randn(6, cols, generator=g)
        values, indices, tail = _teacher(z, 16, 1.0, rest, g)
        z[1], z[4] = NAN, INF
        values[4] = NAN
        weight = torch.tensor([1.0, 0.0, 0.5, 2.0, 0.0, 1.0])
        _check_loss(z.nan_to_num(0.0, 0.0, 0.0) * (weight[:, None] != 0), values.nan_to_num(0.0), indices, tail, 1.0, weight)
        zd = z.to(DEV).requires_grad_()
        out = distill_loss(zd, values.to(DEV), indices.to(DEV), tail=None if tail is None else tail.to(DEV), row_weight=weight.to(DEV))
        grad, = torch.autograd.grad(out, zd)
        assert torch.isfinite(out) and torch.isfinite(grad).all() and float(grad[[1, 4]].abs().sum()) == 0
        zd = z.to(DEV).requires_grad_()
        out = distill_loss(zd, values.to(DEV), indices.to(DEV), row_weight=torch.zeros(6, device=DEV))
        assert float(out.detach()) == 0 and float(torch.autograd.grad(out, zd)[0].abs().sum()) == 0


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('cols', [500, 20000])
def test_unused_doubled_and_empty_entries(rest, cols):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(7, cols, generator=g)
    values, indices, tail = _teacher(z, 12, 1.0, rest, g)
    indices[0, 4:] = -1                     # fewer entries than k
    indices[1, 5] = indices[1, 2]           # the same column twice, and three times
    indices[2, 1:3] = indices[2, 0]
    values[3] = -INF                        # only the rest, or nothing
    indices[4] = -1
    values[5, 3:] = -INF
    if tail is not None:
        tail[4] = -INF                      # nothing at all
        tail[6] = -INF                      # no rest
    _check_loss(z, values, indices, tail, 1.0)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
def test_masked_columns_and_wide_gaps(rest, dtype):
    g = torch.Generator().manual_seed(5)
    cols = 1500
    z = torch.randn(6, cols, generator=g)
    for mask in (-INF, LOWEST[dtype]):
        m = z.clone()
        m[0, 300:] = mask                   # the student's mask; the teacher lists what is left
        m[1, ::2] = mask
        m[2, 40] += 400.0                   # one column holds everything
        m[3] += 300.0                       # far from zero
        m[4] -= 300.0
        values, indices, tail = _teacher(torch.where(m.abs() > 1e4, torch.full((), -1e4), m), 8, 1.0, rest, g)
        _check_loss(m.to(dtype), values, indices, tail, 1.0)


def test_rows_that_cannot_be_answered_are_nan_alone():
    g = torch.Generator().manual_seed(6)
    z = torch.randn(6, 700, generator=g)
    values, indices, tail = _teacher(z, 9, 1.0, True, g)
    indices[1, 3] = 700                     # no such column
    z[2, 11] = NAN
    values[3, 2] = NAN
    values[5, 2] = INF                      # softmax of an infinity
    z[4] = -INF
    for t in (None, tail):
        zd = z.to(DEV).requires_grad_()
        rows = distill_loss(zd, values.to(DEV), indices.to(DEV), tail=None if t is None else t.to(DEV), reduction='none')
        grad, = torch.autograd.grad(rows.sum(), zd)
        nan = torch.isnan(rows).cpu().tolist()
        assert nan == [False, True, True, True, True, True]
        assert torch.isfinite(grad[0]).all() and torch.isnan(grad[[1, 3, 5]]).all()


def test_a_listed_column_that_the_student_excludes_costs_everything():
    z = torch.zeros(1, 600)
    z[0, 5] = -INF
    v, i = torch.tensor([[1.0, 0.5]]), torch.tensor([[5, 6]])
    assert float(distill_loss(z.to(DEV), v.to(DEV), i.to(DEV))) == INF
    v[0, 0] = -INF                          # ... unless the teacher gives it nothing
    assert math.isfinite(float(distill_loss(z.to(DEV), v.to(DEV), i.to(DEV))))


def test_slices_and_leading_dimensions():
    g = torch.Generator().manual_seed(7)
    z = torch.randn(5, 3001, generator=g)
    values, indices, tail = _teacher(z, 20, 1.0, True, g)

    def odd(t):
        wide = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)
        wide[:, 1:-2] = t
        return wide[:, 1:-2]
    for dtype in (F32, BF16):
        _check_loss(z.to(dtype), values, indices, tail, 1.0, lay=odd)
        _check_loss(z.to(dtype), values, indices, tail, 1.0, lay=lambda t: t.t().contiguous().t())
    flat = distill_loss(z.to(DEV), values.to(DEV), indices.to(DEV), tail=tail.to(DEV), reduction='none')
    deep = distill_loss(z.view(5, 1, 1, -1).to(DEV), values.view(5, 1, 1, -1).to(DEV), indices.view(5, 1, 1, -1).to(DEV), tail=tail.view(5, 1, 1).to(DEV), reduction='none')
    assert deep.shape == (5, 1, 1) and torch.equal(deep.view(5), flat)
    one = distill_loss(z[0].to(DEV), values[0].to(DEV), indices[0].to(DEV), tail=tail[0].to(DEV))
    assert one.shape == () and float(one) == float(flat[0])
    for shape in ((0, 700), (2, 0, 700)):
        zd = torch.zeros(shape, device=DEV, requires_grad=True)
        out = distill_loss(zd, torch.zeros(shape[:-1] + (4,), device=DEV), torch.zeros(shape[:-1] + (4,), dtype=torch.long, device=DEV))
        assert float(out.detach()) == 0 and torch.autograd.grad(out, zd)[0].shape == torch.Size(shape)


def test_formulas_are_the_derivatives():
    """the reference's gradient against autograd through the definition and against differences, 64 bits, on the CPU"""
    g = torch.Generator().manual_seed(11)
    z = torch.randn(3, 12, generator=g)
    values, indices, tail = _teacher(z, 4, 0.7, True, g)
    indices[1, 2] = indices[1, 0]
    for t in (None, tail):
        for r in range(3):
            def total(row):
                u = row / 0.7
                parts = values[r].double() / 0.7 if t is None else torch.cat([values[r].double() / 0.7, t[r:r + 1].double()])
                lp = parts - torch.logsumexp(parts, 0)
                lq = u - torch.logsumexp(u, 0)
                res = (lp[:4].exp() * (lp[:4] - lq[indices[r]])).sum()
                if t is not None:
                    rest = [j for j in range(12) if j not in indices[r].tolist()]
                    res = res + lp[4].exp() * (lp[4] - torch.logsumexp(lq[rest], 0))
                return 0.49 * res
            leaf = z[r].double().requires_grad_()
            want, = torch.autograd.grad(total(leaf), leaf)
            loss, grad, _, _, _ = _loss_reference(z, values, indices, t, 0.7, torch.ones(3).double(), torch.ones(3).double())
            assert torch.allclose(grad[r], want, rtol=1e-9, atol=1e-12) and abs(float(loss[r] - total(z[r].double()))) < 1e-12
            for j in range(12):
                e = torch.zeros(12, dtype=torch.float64)
                e[j] = 1e-6
                assert abs(float(total(z[r].double() + e) - total(z[r].double() - e)) / 2e-6 - float(want[j])) < 1e-8


# ---------------------------------------------------------------------------------------------------------------- how it is called
def _pass(z, teacher, k, tau, weight=None):
    values, indices, tail = top_logits(teacher, k, temperature=tau)
    leaf = z.detach().requires_grad_()
    loss = distill_loss(leaf, values, indices, tail=tail, temperature=tau, row_weight=weight)
    return [values, indices, tail, loss.detach(), torch.autograd.grad(loss, leaf)[0]]


@pytest.mark.parametrize('rows,cols', [(40, 9001), (2, 100000)])
def test_same_bits_every_time_and_on_other_streams(rows, cols):
    g = torch.Generator().manual_seed(12)
    z, teacher = (torch.randn(rows, cols, generator=g).to(BF16).to(DEV) for _ in range(2))
    first = _pass(z, teacher, 50, 2.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        res = []
        for s in streams:
            with torch.cuda.stream(s):
                res.append(_pass(z, teacher, 50, 2.0))
        torch.cuda.synchronize()
        for r in res:
            assert all(torch.equal(a, b) for a, b in zip(first, r))


@pytest.mark.parametrize('rows,cols', [(20, 9001), (2, 100000)])
def test_captured_and_replayed(rows, cols):
    g = torch.Generator().manual_seed(13)
    z, teacher = (torch.randn(rows, cols, generator=g).to(DEV) for _ in range(2))
    weight = torch.ones(rows, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _pass(z, teacher, 30, 0.5, weight)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(z, teacher, 30, 0.5, weight)
    for i in range(4):
        z.copy_(torch.randn(rows, cols, generator=g))
        teacher.copy_(torch.randn(rows, cols, generator=g))
        weight[i % rows] = float(i)
        graph.replay()
        torch.cuda.synchronize()
        want = _pass(z, teacher, 30, 0.5, weight)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_module_is_the_function():
    g = torch.Generator().manual_seed(14)
    z, teacher = (torch.randn(9, 500, generator=g).to(DEV) for _ in range(2))
    values, indices, tail = top_logits(teacher, 10, temperature=3.0)
    m = TopLogitsDistillLoss(temperature=3.0, reduction='sum')
    assert torch.equal(m(z, values, indices, tail=tail), distill_loss(z, values, indices, tail=tail, temperature=3.0, reduction='sum'))


def test_teacher_against_itself_costs_nothing():
    """a student that is the teacher: the loss is 0 and so is the gradient, to the roundings of a row"""
    g = torch.Generator().manual_seed(15)
    z = torch.randn(8, 8192, generator=g).mul(4).to(DEV)
    values, indices, tail = top_logits(z, 64, temperature=0.5)
    leaf = z.clone().requires_grad_()
    loss = distill_loss(leaf, values, indices, tail=tail, temperature=0.5)
    grad, = torch.autograd.grad(loss, leaf)
    err = U24 * (8 * 64 + 64 + 32)          # u spans less than 64 here
    assert abs(float(loss.detach())) <= 0.25 * 3 * err and float(grad.abs().sum()) <= 2 * 0.5 * 3 * err


def test_no_second_derivative():
    z = torch.randn(3, 64, device=DEV, requires_grad=True)
    loss = distill_loss(z, *top_logits(z.detach(), 4)[:2])
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(loss, z, create_graph=True)


def test_more_than_2_31_elements():
    """rows do not know of each other: those at the end of a large tensor are the rows of a small call (of as many whole workgroups a row), bit for bit"""
    rows, cols, k = 20000, 131072, 40                              # 2.6e9 elements
    g = torch.Generator(device=DEV).manual_seed(23)
    z = torch.randn((rows, cols), generator=g, device=DEV, dtype=BF16)
    pick = torch.cat([torch.arange(0, 400), torch.arange(16300, 16484), torch.arange(rows - 100, rows)]).to(DEV)          # more rows than are cut
    res = []
    for some in (None, pick):
        zs = z if some is None else z[some]
        values, indices, tail = top_logits(zs, k)
        leaf = zs.detach().requires_grad_()
        loss = distill_loss(leaf, values * 0.5, indices, tail=tail, reduction='none')
        grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        res.append([v if some is not None else v[pick] for v in (values, indices, tail, loss.detach(), grad)])
        del grad, loss, leaf
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_modes_around_the_call():
    z, t = torch.randn(4, 300, device=DEV), torch.randn(4, 300, device=DEV)
    with torch.inference_mode():
        values, indices, tail = top_logits(t, 5)
        a = distill_loss(z, values, indices, tail=tail)
    values, indices, tail = top_logits(t, 5)
    leaf = z.clone().requires_grad_()
    b = distill_loss(leaf, values, indices, tail=tail)
    assert torch.equal(a, b.detach()) and not a.requires_grad
    b.backward()
    with pytest.raises(RuntimeError, match='second time'):
        b.backward()
    c = distill_loss(leaf, values, indices, tail=tail)
    values.mul_(2.0)                                                # a saved tensor is changed before the backward pass
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        c.backward()
    weight = torch.tensor([True, False, True, True], device=DEV)
    d = distill_loss(z, values, indices, row_weight=weight)
    assert torch.equal(d, distill_loss(z, values, indices, row_weight=weight.float()))


def test_two_graphs_at_once_share_nothing():
    """two captured calls, replayed on two streams at the same time"""
    g = torch.Generator().manual_seed(25)
    zs = [torch.randn(3, 100000, generator=g).to(DEV) for _ in range(2)]
    graphs, outs = [], []
    for z in zs:
        _pass(z, z, 20, 1.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_pass(z, z.flip(0), 20, 1.0))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        for z in zs:
            z.copy_(torch.randn(3, 100000, generator=g))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for z, out in zip(zs, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, _pass(z, z.flip(0), 20, 1.0)))


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('cols', [2, 25, 660, 9000, 70001])
def test_logits_far_from_zero_at_a_small_temperature(cols, rest, dtype):
    """the loss depends on differences: a row that is moved as a whole loses no digits (constant, close together, rising by thousands of widths)"""
    g = torch.Generator().manual_seed(cols)
    k = min(cols, 17)
    z = torch.stack([torch.full((cols,), -60.0), torch.full((cols,), 60.0), -60.0 + 0.1 * torch.randn(cols, generator=g), 91.7 + 0.1 * torch.randn(cols, generator=g),
                     torch.linspace(-60.5, -59.5, cols), torch.linspace(61.0, 60.0, cols)]).to(dtype)
    for tau in (0.07, 0.3):
        values, indices, tail = _teacher(z, k, tau, rest, g)
        _check_loss(z, values, indices, tail, tau)


@pytest.mark.parametrize('cols', [30, 20000, 70001])
def test_the_tail_alone_wherever_it_lies(cols):
    """no entry is used: the teacher says 'one of all columns' however large or small its tail's logarithm; listed values of -inf beside it count nothing"""
    g = torch.Generator().manual_seed(cols)
    z = torch.randn(6, cols, generator=g)
    tail = torch.tensor([-846.0, -3e5, -1.0, 0.0, 700.0, 4e6])
    values, indices = torch.randn(6, 3, generator=g), torch.full((6, 3), -1)
    indices[1, 0], values[1, 0] = 7, -INF
    indices[4, 1], values[4, 1] = 7, -INF
    for tau in (0.07, 1.0):
        _check_loss(z, values, indices, tail, tau)
    got = distill_loss(z.to(DEV), values.to(DEV), indices.to(DEV), tail=tail.to(DEV), reduction='none')
    assert float(got[[0, 2, 3, 5]].abs().max()) <= 1e-5                     # nothing is left out: -log(all of it)


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('cols', [8, 3000, 70001])
def test_lowest_values_as_masks_at_every_temperature(cols, rest, dtype):
    """columns that the student masks with its type's lowest value or -inf: few, most, whole stretches of a row, all that are not listed"""
    g = torch.Generator().manual_seed(cols)
    k = 3
    for mask in (LOWEST[dtype], -INF):
        for tau in (0.07, 1.0, 4.0, 50.0):
            z = torch.randn(5, cols, generator=g).to(dtype)
            values, indices, tail = _teacher(z, k, tau, rest, g)
            out = torch.rand(5, cols, generator=g) < torch.tensor([0.05, 0.5, 0.95, 0.0, 1.0])[:, None]
            out[3, cols // 4:] = True
            out.scatter_(1, indices, False)
            z[out] = mask
            if rest:
                tail[4] = -INF                                      # (the teacher's whole mass is listed, as the student's)
            if mask == -INF:
                _check_loss(z, values, indices, tail, tau)
                continue
            # a probability under the smallest float is 0: bit for bit what -inf gives, unless nothing unlisted is left of a row that needs it
            res = []
            for m in (mask, -INF):
                zd = z.masked_fill(out, m).to(DEV).requires_grad_()
                loss = distill_loss(zd, values.to(DEV), indices.to(DEV), tail=tail.to(DEV) if rest else None, temperature=tau, reduction='none')
                res.append((loss.detach().cpu(), torch.autograd.grad(loss.sum(), zd)[0].cpu()))
            nothing = out.sum(1) == cols - k
            same = ~nothing if rest else torch.ones(5, dtype=torch.bool)
            if rest:
                same[4] = True
            if dtype == F16 and tau > 1.0:                          # (its lowest value over such a temperature is not that low)
                _check_loss(z, values, indices, tail, tau)
                continue
            assert torch.equal(res[0][0][same], res[1][0][same]) and torch.equal(res[0][1][same], res[1][1][same])
            if (~same).any():                                       # finite where float32 can hold it: tau p_t |lowest|, p_t right to a few times 2^-24 |u|
                want = _loss_reference(z, values, indices, tail, tau, torch.ones(5), torch.ones(5))[0][~same]
                big = want > torch.finfo(F32).max
                got = res[0][0][~same].double()
                assert bool((got[big] == INF).all()) and bool(((got - want).abs() <= 1e-4 * want)[~big].all())
                assert not res[0][1].isnan().any()


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('rows,cols,k', [(8197, 100, 64), (8200, 600, 8), (8193, 7, 7), (8209, 1, 1), (1201, 4800, 256), (501, 2000, 3), (4099, 256, 16), (4100, 8193, 20)])
def test_many_short_rows(rows, cols, k, rest, dtype):
    """rows that share a wave or hold one alone, the last group not full: padded rows, unused entries, columns named twice, slices at any address"""
    g = torch.Generator().manual_seed(rows + cols)
    z = (torch.randn(rows, cols, generator=g) * 2).to(dtype)
    values, indices, tail = _teacher(z, k, 0.5, rest, g)
    if k > 2:
        indices[::3, 1] = indices[::3, 0]
        indices[1::5, 2] = -1
    weight = torch.rand(rows, generator=g) / 64 * (torch.rand(rows, generator=g) < 0.8)         # (fp16 gradients of 'sum' stay in range)
    _check_loss(z, values, indices, tail, 0.5, weight, lay=lambda t: torch.nn.functional.pad(t, (3, 2))[:, 3:3 + cols])


def test_short_rows_beyond_2_31_elements():
    rows, cols, k = 2200000, 1000, 4
    g = torch.Generator(device=DEV).manual_seed(29)
    z = torch.randn((rows, cols), generator=g, device=DEV, dtype=BF16)
    pick = torch.cat([torch.arange(0, 8192), torch.arange(rows - 300, rows)]).to(DEV)
    res = []
    for some in (None, pick):
        zs = z if some is None else z[some]
        values, indices, tail = top_logits(zs, k)
        leaf = zs.detach().requires_grad_()
        loss = distill_loss(leaf, values * 0.5, indices, tail=tail, reduction='none')
        grad, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        res.append([v if some is not None else v[pick] for v in (values, indices, tail, loss.detach(), grad)])
        del grad, loss, leaf
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rows,cols,ks', [(3, 64, (1, 32, 64)), (70, 65, (5, 33, 65)), (1025, 300, (3, 32, 64, 130)), (2050, 2047, (16, 60, 190)), (1100, 513, (32, 256)),
                                          (300, 4097, (96, 128)), (8200, 40, (7, 40))])
def test_top_logits_of_short_rows(rows, cols, ks, dtype):
    """a wave to eight waves a row: values with many equal ones, masks, NaN, rows at any address"""
    g = torch.Generator().manual_seed(rows + cols)
    z = torch.randn(rows, cols + 5, generator=g) * 3
    z[1::7] = z[1::7].round()                       # a few distinct values
    z[2::11] = (z[2::11] > 3).float()
    z[2, :cols // 2] = -INF
    z[0, 7:] = LOWEST[dtype]
    z[5 % rows, 9::3] = INF
    z[6 % rows, 11] = NAN
    z = z.to(dtype).to(DEV)[:, 3:3 + cols]
    for k in ks:
        _check_top(z, k, 0.5)


@pytest.mark.parametrize('rows,cols', [(9000, 300), (700, 900)])
def test_short_rows_captured_and_on_other_streams(rows, cols):
    g = torch.Generator().manual_seed(rows)
    z, t = (torch.randn(rows, cols, generator=g).to(DEV) for _ in range(2))
    _pass(z, t, 20, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(z, t, 20, 1.0)
    for i in range(3):
        z.copy_(torch.randn(rows, cols, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = _pass(z, t, 20, 1.0)
        side.synchronize()
        want = _pass(z, t, 20, 1.0)
        assert all(torch.equal(a, b) and torch.equal(b, c) for a, b, c in zip(out, want, other))


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('apart', [0.5, 0.02])
@pytest.mark.parametrize('rows,cols,k,tau,each', [(3, 168911, 1, 4.0, 16), (2, 33007, 2, 2.0, 16), (356, 2950, 213, 4.0, 48), (40, 30000, 64, 2.0, 64), (8200, 100, 4, 4.0, 8),
                                                  (600, 12001, 8, 8.0, 32)])
def test_a_student_close_to_its_teacher(rows, cols, k, tau, each, apart, dtype):
    """the loss is of second order in the difference of the two distributions, with p_l and q_l their listed mass about tau^2 (p_l - q_l)^2 / 2 p_l: no error of the first order may
    enter it.  The streamed sum s is off by E relative: 3 roundings of an exponent of at most the row's span, twice (the running maximum's factors), 2 of an
    exponential, `each` columns a thread with half as many roundings for the factors, the joins of lanes, waves and pieces (64 are enough).  It moves
    q_l by q_l q_t E and, both distributions being of sum 1, the loss by tau^2 (|p_l - q_l| E + q_l E^2).  An unlisted column's gradient (q_t - p_t) r, r = exp / s, is
    off by r q_l E and E relative for its own quotient, a listed one's q - p by E q, both by their exponentials' roundings and 16 of the factors."""
    g = torch.Generator().manual_seed(rows + cols)
    z = torch.randn(rows, cols, generator=g).mul(3).to(dtype)
    t = z.double() + apart * torch.randn(rows, cols, generator=g).double()
    v, i = torch.sort(t, dim=1, descending=True)
    tail = torch.logsumexp(v[:, k:] / tau, 1).float()
    values, indices = v[:, :k].to(dtype), i[:, :k].contiguous()
    del t, v, i
    zd = z.to(DEV).requires_grad_()
    got = distill_loss(zd, values.to(DEV), indices.to(DEV), tail=tail.to(DEV), temperature=tau, reduction='none')
    scale = 2.0 ** 12                                               # (fp16 gradients in range)
    grad, = torch.autograd.grad(got, zd, torch.full((rows,), scale, device=DEV))
    u, uv = z.double() / tau, values.double() / tau
    lp = torch.log_softmax(torch.cat([uv, tail.double()[:, None]], 1), 1)
    lse = torch.logsumexp(u, 1, keepdim=True)
    rest = u.scatter(1, indices, -INF)
    lrest = torch.logsumexp(rest, 1, keepdim=True)
    lq = torch.cat([torch.gather(u, 1, indices) - lse, lrest - lse], 1)
    p, q = lp.exp(), lq.exp()
    want = tau ** 2 * (p * (lp - lq)).sum(1)
    span, pl, ql = u.amax(1) - u.amin(1), p[:, :k].sum(1), q[:, :k].sum(1)
    E = U24 * (6 * span + 2 * each + 64)
    tol = tau ** 2 * ((pl - ql).abs() * E + ql * E * E) + 2 * U24 * want.abs()
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= tol).all()), (float((off / want).max()), float((off / tol).max()))
    r = (rest - lrest).exp()
    want = r * (q[:, k:] - p[:, k:])
    tol = r * (ql * E)[:, None] + want.abs() * (E + U24 * (3 * span + 16))[:, None]
    vspan = uv.amax(1) - uv.amin(1)
    want.scatter_(1, indices, q[:, :k] - p[:, :k])
    tol.scatter_(1, indices, (q + p)[:, :k] * (E + U24 * (3 * (span + vspan) + 16))[:, None])
    tol = scale * tau * (tol + STEP[dtype] * (want.abs() + tol)) + (2.0 ** -25 if dtype == F16 else 2.0 ** -126) + 2 * scale * tau * 2.0 ** -126
    off = (grad.double().cpu() - scale * tau * want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('rows,cols', [(4, 3), (40, 100), (8200, 3), (40, 700), (40, 9000), (2, 70001)])
def test_nan_beside_nothing_but_masked_columns(rows, cols, dtype):
    """one unlisted column is NaN and every other unlisted one -inf, in the whole row or in its piece's part alone: softmax of such a row is NaN"""
    k = 2
    g = torch.Generator().manual_seed(cols)
    for place in (0, cols // 2, cols - 1):
        for alone in (True, False):
            z = torch.randn(rows, cols, generator=g)
            free = [j for j in range(cols) if j != place]
            listed = torch.tensor([free[0], free[-1]])
            if alone:
                keep = z[0, listed].clone()
                z[0] = -INF
                z[0, listed] = keep
            z[0, place] = NAN
            values, indices = torch.randn(rows, k, generator=g), listed.expand(rows, k)
            for tail in (0.3, -INF, None):
                zd = z.to(dtype).to(DEV).requires_grad_()
                out = distill_loss(zd, values.to(DEV), indices.to(DEV), tail=None if tail is None else torch.full((rows,), tail, device=DEV), reduction='none')
                grad, = torch.autograd.grad(out.sum(), zd)
                assert out.isnan().tolist() == [True] + [False] * (rows - 1), (place, alone, tail, float(out[0]))
                assert grad[0].isnan().all() and grad[1:].isfinite().all(), (place, alone, tail)


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=str)
@pytest.mark.parametrize('rows,cols,k', [(2000, 3000, 64), (600, 9000, 128), (300, 20000, 256)])
def test_top_logits_of_many_rows_without_a_finite_bound(rows, cols, k, dtype):
    """rows of which masks leave fewer than k columns, or with more than k infinities: the search for a bound runs twice over all waves"""
    g = torch.Generator().manual_seed(cols)
    z = torch.full((rows, cols), -INF)
    for r in range(rows):
        at = torch.randint(0, cols, (k - 3,), generator=g)
        z[r, at] = torch.randn(k - 3, generator=g)
    z[::3] = torch.randn(len(z[::3]), cols, generator=g)
    z[::3].masked_fill_(torch.rand(len(z[::3]), cols, generator=g) < 2.0 * k / cols, INF)
    z = z.to(dtype).to(DEV)
    _check_top(z, k, 1.0)


# A launch has fewer than 2^32 threads: calls of more rows go in parts.  Rows overlap in memory (row r begins at element r), so that many of them take little.
def _overlapping(rows, cols, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(rows + cols, generator=g, device=DEV).mul(2).to(dtype).as_strided((rows, cols), (1, 1))


def _about(rows, border):
    return torch.tensor(sorted({r for b in (0, border, rows) for r in range(b - 4, b + 4) if 0 <= r < rows}), device=DEV)


@pytest.mark.parametrize('rows,cols,k,threads', [(2 ** 26 + 9, 8, 1, 64), (2 ** 23 + 9, 300, 256, 512)])
def test_top_logits_of_more_rows_than_a_launch_holds(rows, cols, k, threads):
    z = _overlapping(rows, cols, BF16, 41)
    pick = _about(rows, 0xffffff00 // threads // 16 * 16)
    values, indices, tail = top_logits(z, k)
    order, want = _top_reference(z[pick].cpu(), k, 1.0)
    assert torch.equal(indices[pick].cpu(), order) and torch.equal(values[pick].cpu(), torch.gather(z[pick].cpu(), 1, order))
    # (logarithms of up to 299 numbers of at most 2 x 6 widths: the tolerance of _check_top at its largest)
    assert float((tail[pick].double().cpu() - want).abs().max()) <= U24 * (8 * 12 + 64 + 2 + 18)


@pytest.mark.parametrize('rows,cols,threads,train', [(2 ** 28 + 9, 8, 16, True), (2 ** 23 + 9, 4100, 512, True), (2 ** 23 + 9, 16400, 512, False)])
@pytest.mark.parametrize('rest', [False, True])
def test_loss_of_more_rows_than_a_launch_holds(rows, cols, threads, train, rest):
    z = _overlapping(rows, cols, BF16, 42).detach().requires_grad_(train)
    values = _overlapping(rows, 1, BF16, 43)
    indices = torch.remainder(torch.arange(rows, dtype=torch.int32, device=DEV), cols)[:, None]
    tail = torch.zeros(rows, device=DEV) if rest else None
    weight = torch.ones(rows, device=DEV)
    weight[::3] = 0.5
    got = distill_loss(z, values, indices, tail=tail, row_weight=weight, reduction='none')
    pick = _about(rows, 0xffffff00 // threads // 16 * 16)
    part = lambda t: None if t is None else t.detach()[pick].cpu()
    one = torch.ones(len(pick), dtype=torch.float64)
    loss, want, mag, err, tiny = _loss_reference(part(z), part(values), part(indices), part(tail), 1.0, part(weight).double(), one)
    assert bool(((part(got).double() - loss).abs() <= 3 * err + 16 * U24 * loss.abs()).all())
    if not train:
        return
    up = torch.ones(rows, device=DEV)
    grad, = torch.autograd.grad(got, z, up)
    step = STEP[BF16]
    tol = (step * want.abs() + 3 * err[:, None] * mag) * (1 + step) + 2.0 ** -126 + tiny
    assert bool(((part(grad).double() - want).abs() <= tol).all())
    if cols > 8:
        return
    total = distill_loss(z, values, indices, tail=tail, row_weight=weight, reduction='sum')
    whole = got.detach().sum(dtype=torch.float64)
    assert abs(float(total.detach()) - float(whole)) <= 2 * U24 * float(whole)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('cols', [3, 700, 9000, 70001])
def test_a_probability_under_the_smallest_float_counts_as_zero(cols, rest):
    """... relative to the largest of its row, whatever the student gives the column: where p = 2^-125 meets q = 0 the loss is infinite, where p = 2^-128 does it is what -inf leaves"""
    z = torch.zeros(3, cols)
    z[:, 1] = -INF
    values, indices = torch.zeros(3, 2), torch.tensor([0, 1]).expand(3, 2)
    values[:, 1] = torch.tensor([-125.0, -128.0, -INF]) * math.log(2.0)
    tail = torch.full((3,), -1.0, device=DEV) if rest else None
    # (with the rest the other probability is 1 / (1 + e^-1): the exponent of p falls by 0.46)
    got = distill_loss(z.to(DEV), values.to(DEV), indices.to(DEV), tail=tail, reduction='none').cpu()
    assert float(got[0]) == INF and math.isfinite(float(got[1])) and torch.equal(got[1], got[2])
