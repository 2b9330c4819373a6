"""The joint between two residual blocks on the HIP path: the norm behind a block, its gate, the residual scale, the skip connection and the norm
in front of the next block - one launch forward, two backward (csrc/residual_norm.hip).

The reference's residual blocks scale their branch (``res += x`` after ``.mul(res_scale)``, rumpy/SISR/models/advanced/common.py:72-73) or gate it per
channel (``CALayer``, architectures.py:41-44, 83); networks with norms around such a block - layer or root-mean-square norm over the channels of a
pixel or token, before the block, after it, or both - need, between two blocks,

    z = N_post(branch)                      y = x + scale * gate * z                      h = N_pre(y)

with y the residual stream and h the next block's input.  ``residual_norm`` is that as a function, ``ResidualNorm`` as a module.
No CPU path: tensors must be on the GPU."""
import functools

import torch
from torch import nn

from rumpy_amd import _lib as L

_FMT = {torch.float32: L.FMT_F32, torch.bfloat16: L.FMT_BF16, torch.float16: L.FMT_F16}
_KIND = {None: 0, 'layer': 1, 'rms': 2}
MAX_CHANNELS = 8192
_GATE_NONE, _GATE_GROUP, _GATE_FULL = 0, 1, 2


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t as rows of contiguous channels: (tensor, row stride in elements); copied only when its rows do not lie at one stride"""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, c
    if t.stride(-1) == 1:
        if t.dim() == 2:
            return t, t.stride(0)
        try:
            return t, t.view(-1, c).stride(0)
        except RuntimeError:
            pass
    return t.contiguous(), c


_raw_stream = torch._C._cuda_getCurrentRawStream          # torch.cuda.current_stream builds a Stream object first: 2 us a call


def _launch(name, args, dev):
    """on the current stream of the tensors' own device, whichever device is current"""
    if dev.index == torch.cuda.current_device():
        L.call(name, args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            L.call(name, args, _raw_stream(dev.index))


def _new_like(t):
    """an uninitialised contiguous tensor of t's shape and type (empty_like is half the price of empty, and keeps strides)"""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@functools.lru_cache(maxsize=512)
def _partial_floats(rows, group_rows, c, gate_mode):
    return int(L.lib().rumpy_residual_norm_partial_floats(rows, group_rows, c, gate_mode))


def _forward(x, branch, gate, post_w, post_b, pre_w, pre_b, cfg, keep):
    """-> (y or None, h or None, stats or None)"""
    post, pre, gate_mode, group_rows, scale, eps = cfg
    c = x.shape[-1]
    rows = x.numel() // c
    tb = x if branch is None else branch
    y = _new_like(x) if branch is not None else None
    h = _new_like(tb) if pre else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if keep else None
    if rows == 0:
        return y, h, stats
    x, ldx = _rows(x)
    ldt = ldg = 0
    if branch is not None:
        branch, ldt = _rows(branch)
    if gate_mode == _GATE_FULL:
        gate, ldg = _rows(gate)
    elif gate is not None:
        gate = gate.contiguous()
    _launch('rumpy_residual_norm_fwd', L.ResidualNormArgs(
        x=x.data_ptr(), t=_p(branch), gate=_p(gate), post_w=_p(post_w), post_b=_p(post_b), pre_w=_p(pre_w), pre_b=_p(pre_b), y=_p(y), h=_p(h),
        stats=_p(stats), rows=rows, group_rows=group_rows, ldx=ldx, ldt=ldt, ldg=ldg, C=c, x_fmt=_FMT[x.dtype], t_fmt=_FMT[tb.dtype],
        gate_mode=gate_mode, post=post, pre=pre, scale=scale, eps=eps), x.device)
    return y, h, stats


def _once_differentiable(name):
    if torch.is_grad_enabled():             # (only under create_graph=True)
        raise RuntimeError('rumpy_amd: %s has no second derivative' % name)


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, post_w, post_b, pre_w, pre_b, cfg):
        y, h, stats = _forward(x, branch, gate, post_w, post_b, pre_w, pre_b, cfg, True)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, branch, gate, post_w, post_b, pre_w, stats)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        _once_differentiable('residual_norm')
        x, branch, gate, post_w, post_b, pre_w, stats = ctx.saved_tensors
        post, pre, gate_mode, group_rows, scale, _ = ctx.cfg
        need = ctx.needs_input_grad
        if dy is None and dh is None:
            return (None,) * 8
        c, dev = x.shape[-1], x.device
        rows = x.numel() // c
        tb = x if branch is None else branch
        dx = _new_like(x) if need[0] else None
        dt = _new_like(branch) if need[1] else None
        dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if need[2] else None
        # (where nothing arrives through the norm in front, its parameters have no gradient)
        wanted = (need[3], need[4], need[5] and dh is not None, need[6] and dh is not None)
        params = torch.empty((4, c), dtype=torch.float32, device=dev).unbind(0) if any(wanted) else (None,) * 4
        d_post_w, d_post_b, d_pre_w, d_pre_b = (p if w else None for p, w in zip(params, wanted))
        if rows == 0:
            for t in (dgate, d_post_w, d_post_b, d_pre_w, d_pre_b):
                if t is not None:
                    t.zero_()
        if rows:
            x, ldx = _rows(x)
            ldt = ldg = lddy = lddh = 0
            if branch is not None:
                branch, ldt = _rows(branch)
            if gate_mode == _GATE_FULL:
                gate, ldg = _rows(gate)
            elif gate is not None:
                gate = gate.contiguous()
            if dy is not None:
                dy, lddy = _rows(dy)
            if dh is not None:
                dh, lddh = _rows(dh)
            partial = torch.empty(_partial_floats(rows, group_rows, c, gate_mode), dtype=torch.float32, device=dev)
            _launch('rumpy_residual_norm_bwd', L.ResidualNormBwdArgs(
                dy=_p(dy), dh=_p(dh), x=x.data_ptr(), t=_p(branch), gate=_p(gate), post_w=_p(post_w), post_b=_p(post_b), pre_w=_p(pre_w),
                stats=stats.data_ptr(), dx=_p(dx), dt=_p(dt), dgate=_p(dgate), d_post_w=_p(d_post_w), d_post_b=_p(d_post_b), d_pre_w=_p(d_pre_w),
                d_pre_b=_p(d_pre_b), partial=partial.data_ptr(), rows=rows, group_rows=group_rows, lddy=lddy, lddh=lddh, ldx=ldx, ldt=ldt, ldg=ldg,
                C=c, x_fmt=_FMT[x.dtype], t_fmt=_FMT[tb.dtype], gate_mode=gate_mode, post=post, pre=pre, scale=scale), dev)
        return dx, dt, dgate, d_post_w, d_post_b, d_pre_w, d_pre_b, None


def _param(p, name, norm, c, dev):
    if p is None:
        return None
    if norm is None:
        raise ValueError('rumpy_amd: residual_norm has %s but no norm it belongs to' % name)
    if p.shape != (c,) or p.dtype != torch.float32 or p.device != dev:
        raise ValueError('rumpy_amd: residual_norm takes %s as float32 [%d] beside its input, not %s %s' % (name, c, p.dtype, tuple(p.shape)))
    return p if p.is_contiguous() else p.contiguous()


def residual_norm(x, branch=None, gate=None, scale=1.0, post_norm=None, post_weight=None, post_bias=None,
                  pre_norm=None, pre_weight=None, pre_bias=None, eps=1e-5):
    """y = x + scale * gate * N_post(branch) ; h = N_pre(y)  ->  (y, h)

    x, branch    [..., C], C <= 8192: the residual stream and the block's output; both float32, bfloat16 or float16, or x in float32 beside a 16-bit
                 branch.  y has x's type, h the branch's.  branch None: (x, N_pre(x)), the norm in front of the first block.
    gate         None; float32 [C] (a learnt scale per channel); float32 [x.shape[0], C] (one gate per image, as CALayer makes it); or
                 [..., C] like the branch, in its type.
    post_norm, pre_norm   None, 'layer' or 'rms', with weight and bias float32 [C] or None.  pre_norm None: h is None.
    Gradients go to x, branch, gate and the four parameters.  Statistics and sums are float32; y, h and the gradients are rounded once (h is the
    norm of the unrounded y).  Channels that do not lie side by side, or rows at no common stride, are copied first.
    mirrors and joins rumpy/SISR/models/advanced/common.py:71-75 and architectures.py:41-44, 81-84 (``res += x`` around a scaled or gated branch)"""
    for k in (post_norm, pre_norm):
        if k not in _KIND:
            raise ValueError("rumpy_amd: residual_norm knows the norms 'layer' and 'rms', not %r" % (k,))
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError('rumpy_amd: residual_norm takes [..., C] with 1 <= C <= %d, not %s' % (MAX_CHANNELS, tuple(x.shape)))
    c, dev = x.shape[-1], x.device
    gate_mode, group_rows = _GATE_NONE, 0
    if branch is None:
        if gate is not None or post_norm is not None or pre_norm is None:
            raise ValueError('rumpy_amd: residual_norm without a branch is the norm in front alone')
        if x.dtype not in _FMT:
            raise RuntimeError('rumpy_amd: residual_norm takes float32, bfloat16 or float16, not %s' % x.dtype)
    else:
        if branch.shape != x.shape or branch.device != dev:
            raise ValueError('rumpy_amd: residual_norm takes a branch like x, %s, not %s' % (tuple(x.shape), tuple(branch.shape)))
        if x.dtype not in _FMT or branch.dtype not in _FMT or (x.dtype != branch.dtype and x.dtype != torch.float32):
            raise RuntimeError('rumpy_amd: residual_norm takes x and branch in one of float32, bfloat16, float16, or x in float32 beside a 16-bit branch, '
                               'not %s and %s' % (x.dtype, branch.dtype))
        if gate is not None:
            if gate.device != dev:
                raise ValueError('rumpy_amd: residual_norm takes a gate beside x')
            rows = x.numel() // c
            if gate.shape == x.shape and gate.dtype == branch.dtype and not (x.dim() == 1 and gate.dtype == torch.float32):
                gate_mode = _GATE_FULL
            elif gate.dtype == torch.float32 and tuple(gate.shape) == (c,):
                gate_mode, group_rows = _GATE_GROUP, max(rows, 1)
            elif gate.dtype == torch.float32 and x.dim() >= 2 and tuple(gate.shape) == (x.shape[0], c):
                gate_mode, group_rows = _GATE_GROUP, max(rows // max(x.shape[0], 1), 1)
            else:
                raise ValueError('rumpy_amd: residual_norm takes a gate as float32 [C], float32 [%d, C] or like the branch, not %s %s'
                                 % (x.shape[0], gate.dtype, tuple(gate.shape)))
    post_weight, post_bias = _param(post_weight, 'post_weight', post_norm, c, dev), _param(post_bias, 'post_bias', post_norm, c, dev)
    pre_weight, pre_bias = _param(pre_weight, 'pre_weight', pre_norm, c, dev), _param(pre_bias, 'pre_bias', pre_norm, c, dev)
    if not x.is_cuda:
        raise RuntimeError('rumpy_amd: residual_norm runs on an MI355X through the HIP extension; there is no CPU path')
    cfg = (_KIND[post_norm], _KIND[pre_norm], gate_mode, group_rows, float(scale), float(eps))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, branch, gate, post_weight, post_bias, pre_weight, pre_bias)):
        y, h = _ResidualNormFn.apply(x, branch, gate, post_weight, post_bias, pre_weight, pre_bias, cfg)
    else:
        y, h, _ = _forward(x, branch, gate, post_weight, post_bias, pre_weight, pre_bias, cfg, False)
    return (x if branch is None else y), h


class ResidualNorm(nn.Module):
    """``residual_norm`` with its parameters: the joint behind one block and in front of the next.

    post_norm / pre_norm: None, 'layer' or 'rms' (weights ones, biases zeros; ``bias=False``: none; 'rms' has none unless asked).
    channel_scale: a learnt gate per channel that starts at this value (None: no such gate; a gate can then be given per call)."""

    def __init__(self, features, scale=1.0, post_norm=None, pre_norm='layer', bias=None, channel_scale=None, eps=1e-5):
        super(ResidualNorm, self).__init__()
        if not 1 <= features <= MAX_CHANNELS:
            raise ValueError('rumpy_amd: ResidualNorm takes 1 .. %d features, not %r' % (MAX_CHANNELS, features))
        for k in (post_norm, pre_norm):
            if k not in _KIND:
                raise ValueError("rumpy_amd: ResidualNorm knows the norms 'layer' and 'rms', not %r" % (k,))
        self.features, self.scale, self.post_norm, self.pre_norm, self.eps = features, scale, post_norm, pre_norm, eps
        with_bias = lambda kind: kind is not None and (kind == 'layer' if bias is None else bias)
        self.post_weight = nn.Parameter(torch.ones(features)) if post_norm else None
        self.post_bias = nn.Parameter(torch.zeros(features)) if with_bias(post_norm) else None
        self.pre_weight = nn.Parameter(torch.ones(features)) if pre_norm else None
        self.pre_bias = nn.Parameter(torch.zeros(features)) if with_bias(pre_norm) else None
        self.gate = nn.Parameter(torch.full((features,), float(channel_scale))) if channel_scale is not None else None

    def forward(self, x, branch=None, gate=None):
        """-> (y, h) as ``residual_norm``; branch None: (x, h), the norm in front of the first block"""
        if gate is not None and self.gate is not None:
            raise ValueError('rumpy_amd: this ResidualNorm has a gate of its own')
        if branch is None:
            return residual_norm(x, pre_norm=self.pre_norm, pre_weight=self.pre_weight, pre_bias=self.pre_bias, eps=self.eps)
        return residual_norm(x, branch, gate=self.gate if gate is None else gate, scale=self.scale, post_norm=self.post_norm, post_weight=self.post_weight,
                             post_bias=self.post_bias, pre_norm=self.pre_norm, pre_weight=self.pre_weight, pre_bias=self.pre_bias, eps=self.eps)
