"""The joint between two residual blocks on the HIP path: the norm behind a block, its gate, the residual scale, the skip connection and the norm
in front of the next block - one launch forward, two backward (csrc/residual_norm.hip, bound to torch by csrc/torch_bind.cpp).

The reference's residual blocks scale their branch (``res += x`` after ``.mul(res_scale)``, rumpy/SISR/models/advanced/common.py:72-73) or gate it per
channel (``CALayer``, architectures.py:41-44, 83); networks with norms around such a block - layer or root-mean-square norm over the channels of a
pixel or token, before the block, after it, or both - need, between two blocks,

    z = N_post(branch)                      y = x + scale * gate * z                      h = N_pre(y)

with y the residual stream and h the next block's input.  ``residual_norm`` is that as a function, ``ResidualNorm`` as a module.
No CPU path: tensors must be on the GPU."""
import torch
from torch import nn

from rumpy_amd import _lib as L

MAX_CHANNELS = 8192


def residual_norm(x, branch=None, gate=None, scale=1.0, post_norm=None, post_weight=None, post_bias=None,
                  pre_norm=None, pre_weight=None, pre_bias=None, eps=1e-5):
    """y = x + scale * gate * N_post(branch) ; h = N_pre(y)  ->  (y, h)

    x, branch    [..., C], C <= 8192: the residual stream and the block's output; both float32, bfloat16 or float16, or x in float32 beside a 16-bit
                 branch.  y has x's type, h the branch's.  branch None: (x, N_pre(x)), the norm in front of the first block.
    gate         None; float32 [C] (a learnt scale per channel); float32 [x.shape[0], C] (one gate per image, as CALayer makes it); or
                 [..., C] like the branch, in its type.
    post_norm, pre_norm   None, 'layer' or 'rms', with weight and bias float32 [C] or None.  pre_norm None: h is None.
    eps          above zero.
    Gradients go to x, branch, gate and the four parameters.  Statistics and sums are float32; y, h and the gradients are rounded once (h is the
    norm of the unrounded y).  Channels that do not lie side by side, or rows at no common stride, are copied first.
    mirrors and joins rumpy/SISR/models/advanced/common.py:71-75 and architectures.py:41-44, 81-84 (``res += x`` around a scaled or gated branch)"""
    return (L.OPS or L.ops()).residual_norm(x, branch, gate, scale, post_norm, post_weight, post_bias, pre_norm, pre_weight, pre_bias, eps)


class ResidualNorm(nn.Module):
    """``residual_norm`` with its parameters: the joint behind one block and in front of the next.

    post_norm / pre_norm: None, 'layer' or 'rms' (weights ones, biases zeros; ``bias=False``: none; 'rms' has none unless asked).
    channel_scale: a learnt gate per channel that starts at this value (None: no such gate; a gate can then be given per call)."""

    def __init__(self, features, scale=1.0, post_norm=None, pre_norm='layer', bias=None, channel_scale=None, eps=1e-5):
        super(ResidualNorm, self).__init__()
        if not 1 <= features <= MAX_CHANNELS:
            raise ValueError('rumpy_amd: ResidualNorm takes 1 .. %d features, not %r' % (MAX_CHANNELS, features))
        for k in (post_norm, pre_norm):
            if k not in (None, 'layer', 'rms'):
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
