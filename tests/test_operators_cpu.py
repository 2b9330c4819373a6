"""residual_norm, top_logits and distill_loss without a GPU: structures, refusals of the C entry points and of the Python functions."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from rumpy_amd import _lib as L
from rumpy_amd.distill import distill_loss, top_logits
from rumpy_amd.residual_norm import ResidualNorm, residual_norm
from rumpy_amd.sr_tools.loss_functions import TopLogitsDistillLoss

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E_ARG = -1


def _lib_or_skip():
    if not os.path.isfile(L.LIB_PATH):
        pytest.skip('librumpy_amd.so not built')
    return L.lib()


def test_structures_match_the_header(tmp_path):
    pairs = {'rumpy_residual_norm_args': L.ResidualNormArgs, 'rumpy_residual_norm_bwd_args': L.ResidualNormBwdArgs, 'rumpy_top_logits_args': L.TopLogitsArgs,
             'rumpy_distill_args': L.DistillArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "rumpy_amd.h"', 'int main(void){']
    for name, st in pairs.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (name, name))
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (name, f) for f, _ in st._fields_]
        lines.append('printf("\\n");')
    src, exe = tmp_path / 'p.c', tmp_path / 'p'
    src.write_text('\n'.join(lines + ['return 0;}']))
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    for line in subprocess.check_output([str(exe)]).decode().strip().splitlines():
        name, size, *offsets = line.split()
        st = pairs[name]
        assert int(size) == ctypes.sizeof(st)
        assert [getattr(st, f).offset for f, _ in st._fields_] == [int(o) for o in offsets], name


# pointers that no call below follows: every one of these calls is refused on the host
P = 4096


def _norm_args(**kw):
    d = dict(x=P, t=P, y=P, h=P, rows=4, C=64, ldx=64, ldt=64, x_fmt=L.FMT_BF16, t_fmt=L.FMT_BF16, post=1, pre=2, scale=1.0, eps=1e-5)
    d.update(kw)
    return L.ResidualNormArgs(**d)


@pytest.mark.parametrize('bad', [dict(C=0), dict(C=8193), dict(rows=-1), dict(rows=2 ** 31), dict(x=None), dict(y=None), dict(h=None), dict(post=3), dict(pre=-1),
                                 dict(x_fmt=2), dict(t_fmt=L.FMT_F16), dict(x_fmt=L.FMT_BF16, t_fmt=L.FMT_F32), dict(gate_mode=1), dict(gate=P),
                                 dict(gate=P, gate_mode=3), dict(gate=P, gate_mode=1, group_rows=0), dict(gate=P, gate_mode=1, group_rows=3),
                                 dict(t=None, post=1), dict(t=None, post=0, pre=0), dict(t=None, post=0, gate=P, gate_mode=2), dict(ldx=-1)], ids=str)
def test_norm_entry_point_refuses(bad):
    lib = _lib_or_skip()
    assert lib.rumpy_residual_norm_fwd(ctypes.byref(_norm_args(**bad)), None) == E_ARG
    assert b'rumpy_residual_norm_fwd' in lib.rumpy_last_error()


def test_norm_entry_point_takes_no_rows_and_no_arguments():
    lib = _lib_or_skip()
    assert lib.rumpy_residual_norm_fwd(ctypes.byref(_norm_args(rows=0, x=None, t=P, y=None, h=None)), None) == 0
    assert lib.rumpy_residual_norm_fwd(None, None) == E_ARG and lib.rumpy_residual_norm_bwd(None, None) == E_ARG
    assert lib.rumpy_top_logits(None, None) == E_ARG and lib.rumpy_distill_fwd(None, None) == E_ARG and lib.rumpy_distill_bwd(None, None) == E_ARG


@pytest.mark.parametrize('bad', [dict(rows=0), dict(x=None), dict(partial=None), dict(dy=None, dh=None), dict(pre=0), dict(stats=None), dict(dgate=P),
                                 dict(t=None, post=0), dict(post=0, d_post_w=P), dict(dh=None, d_pre_b=P), dict(lddh=-2), dict(C=9000)], ids=str)
def test_norm_backward_entry_point_refuses(bad):
    lib = _lib_or_skip()
    d = dict(dy=P, dh=P, x=P, t=P, stats=P, dx=P, dt=P, partial=P, rows=4, C=64, lddy=64, lddh=64, ldx=64, ldt=64, x_fmt=L.FMT_BF16, t_fmt=L.FMT_BF16, post=1, pre=2,
             scale=1.0)
    d.update(bad)
    assert lib.rumpy_residual_norm_bwd(ctypes.byref(L.ResidualNormBwdArgs(**d)), None) == E_ARG
    assert b'rumpy_residual_norm_bwd' in lib.rumpy_last_error()


@pytest.mark.parametrize('bad', [dict(k=0), dict(k=257), dict(V=9, k=10), dict(V=0), dict(V=2 ** 30 + 1), dict(rows=-1), dict(ld=-1), dict(fmt=2), dict(tau=0.0),
                                 dict(tau=float('inf')), dict(tau=float('nan')), dict(logits=None), dict(values=None), dict(indices=None), dict(tail=None),
                                 dict(V=200000, rows=1), dict(V=200000, rows=1, work=P + 4), dict(rows=2 ** 31)], ids=str)
def test_top_logits_entry_point_refuses(bad):
    lib = _lib_or_skip()
    d = dict(logits=P, values=P, indices=P, tail=P, rows=3, ld=500, V=500, k=10, fmt=L.FMT_F32, tau=1.0)
    d.update(bad)
    assert lib.rumpy_top_logits(ctypes.byref(L.TopLogitsArgs(**d)), None) == E_ARG
    assert b'rumpy_top_logits' in lib.rumpy_last_error()


@pytest.mark.parametrize('bad', [dict(k=0), dict(k=257), dict(V=0), dict(V=2 ** 30 + 1), dict(rows=-1), dict(ld=-1), dict(fmt=2), dict(value_fmt=5), dict(tau=0.0),
                                 dict(tau=float('nan')), dict(tau=-1.0), dict(logits=None), dict(top_values=None), dict(top_indices=None), dict(row_loss=None),
                                 dict(state=None), dict(factor=None), dict(V=200000, partial=None), dict(rows=2 ** 32)], ids=str)
def test_distill_entry_points_refuse(bad):
    lib = _lib_or_skip()
    d = dict(logits=P, top_values=P, top_indices=P, row_loss=P, state=P, loss=P, factor=P, partial=P, gout=P, dlogits=P, rows=3, ld=500, V=500, k=10, fmt=L.FMT_F32,
             value_fmt=L.FMT_F32, index64=1, mean=1, tau=1.0)
    d.update(bad)
    for name in ('rumpy_distill_fwd', 'rumpy_distill_bwd'):
        assert getattr(lib, name)(ctypes.byref(L.DistillArgs(**d)), None) == E_ARG
        assert name.encode() in lib.rumpy_last_error()


def test_workspace_sizes():
    lib = _lib_or_skip()
    assert lib.rumpy_residual_norm_partial_floats(0, 1, 64, 0) == 0 and lib.rumpy_residual_norm_partial_floats(5, 1, 9000, 0) == 0
    for rows, group, c, mode in ((1, 1, 64, 0), (1000, 10, 64, 1), (1000, 500, 64, 1), (100000, 100000, 4096, 1), (7, 1, 8192, 2)):
        n = lib.rumpy_residual_norm_partial_floats(rows, group, c, mode)
        assert n > 0 and n % c == 0
        # at least the four parameters' partial rows, and one partial gate row per gate row
        assert n // c >= 4 + (rows // group if mode == 1 else 0)
    assert lib.rumpy_distill_partial_floats(0, 100000) == 0 and lib.rumpy_distill_partial_floats(4096, 50000) == 0
    assert lib.rumpy_distill_partial_floats(1, 262144) > 0
    assert lib.rumpy_top_logits_work_bytes(1000, 50000, 64) == 0 and lib.rumpy_top_logits_work_bytes(32, 8192, 64) == 0
    assert lib.rumpy_top_logits_work_bytes(1, 262144, 64) > 0 and lib.rumpy_top_logits_work_bytes(1, 262144, 257) == 0


# ---------------------------------------------------------------------------------------------------------------- Python refusals
def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize('call,error,text', [
    (lambda: residual_norm(_t(3, 8), _t(3, 8), post_norm='batch'), ValueError, 'layer'),
    (lambda: residual_norm(_t(3, 8), _t(3, 9), pre_norm='rms'), ValueError, 'branch like x'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8, dtype=torch.bfloat16), gate=_t(3, 8, dtype=torch.float16), pre_norm='rms'), ValueError, 'gate'),
    (lambda: residual_norm(_t(4, 3, 8), _t(4, 3, 8), gate=_t(3, 8), pre_norm='rms'), ValueError, 'gate'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), gate=_t(8, dtype=torch.bfloat16), pre_norm='rms'), ValueError, 'gate'),
    (lambda: residual_norm(_t(3, 8, dtype=torch.float64), _t(3, 8, dtype=torch.float64), pre_norm='rms'), RuntimeError, 'float64'),
    (lambda: residual_norm(_t(3, 8, dtype=torch.bfloat16), _t(3, 8), pre_norm='rms'), RuntimeError, 'float32'),
    (lambda: residual_norm(_t(3, 8, dtype=torch.bfloat16), _t(3, 8, dtype=torch.float16), pre_norm='rms'), RuntimeError, 'float16'),
    (lambda: residual_norm(_t(3, 8193), _t(3, 8193), pre_norm='rms'), ValueError, '8192'),
    (lambda: residual_norm(_t(3, 0), _t(3, 0), pre_norm='rms'), ValueError, '8192'),
    (lambda: residual_norm(_t(()), _t(()), pre_norm='rms'), ValueError, 'C'),
    (lambda: residual_norm(_t(3, 8)), ValueError, 'without a branch'),
    (lambda: residual_norm(_t(3, 8), gate=_t(8), pre_norm='rms'), ValueError, 'without a branch'),
    (lambda: residual_norm(_t(3, 8, dtype=torch.int32), pre_norm='rms'), RuntimeError, 'int32'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), post_weight=_t(8)), ValueError, 'no norm'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), pre_norm='rms', pre_weight=_t(7)), ValueError, 'pre_weight'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), pre_norm='rms', pre_bias=_t(8, dtype=torch.bfloat16)), ValueError, 'pre_bias'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), pre_norm='rms', eps=0.0), ValueError, 'eps'),
    (lambda: residual_norm(_t(3, 8), _t(3, 8), pre_norm='rms'), RuntimeError, 'no CPU path'),
    (lambda: ResidualNorm(0), ValueError, 'features'),
    (lambda: ResidualNorm(8, pre_norm='group'), ValueError, 'layer'),
    (lambda: ResidualNorm(8, channel_scale=1.0)(_t(3, 8), _t(3, 8), gate=_t(8)), ValueError, 'gate of its own'),
    (lambda: top_logits(_t(3, 8), 0), ValueError, 'k'),
    (lambda: top_logits(_t(3, 8), 9), ValueError, 'k'),
    (lambda: top_logits(_t(3, 800), 257), ValueError, '256'),
    (lambda: top_logits(_t(3, 0), 1), ValueError, 'V'),
    (lambda: top_logits(_t(3, 8), 2, temperature=0.0), ValueError, 'temperature'),
    (lambda: top_logits(_t(3, 8), 2, temperature=float('nan')), ValueError, 'temperature'),
    (lambda: top_logits(_t(3, 8, dtype=torch.float64), 2), RuntimeError, 'float64'),
    (lambda: top_logits(_t(3, 8), 2), RuntimeError, 'no CPU path'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 2, dtype=torch.long), reduction='max'), ValueError, 'reduces'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 3, dtype=torch.long)), ValueError, 'top logits'),
    (lambda: distill_loss(_t(3, 8), _t(2, 2), _t(2, 2, dtype=torch.long)), ValueError, 'top logits'),
    (lambda: distill_loss(_t(3, 8), _t(3, 0), _t(3, 0, dtype=torch.long)), ValueError, 'top logits'),
    (lambda: distill_loss(_t(3, 800), _t(3, 257), _t(3, 257, dtype=torch.long)), ValueError, '256'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 2)), RuntimeError, 'int64'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2, dtype=torch.float64), _t(3, 2, dtype=torch.long)), RuntimeError, 'float64'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 2, dtype=torch.long), tail=_t(4)), ValueError, 'tail'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 2, dtype=torch.long), row_weight=_t(3, 1)), ValueError, 'row_weight'),
    (lambda: distill_loss(_t(3, 8), _t(3, 2), _t(3, 2, dtype=torch.long), temperature=-1.0), ValueError, 'temperature'),
    (lambda: TopLogitsDistillLoss()(_t(3, 8), _t(3, 2), _t(3, 2, dtype=torch.long)), RuntimeError, 'no CPU path'),
])
def test_python_refusals(call, error, text):
    with pytest.raises(error, match=re.escape(text)):
        call()


def test_binding_is_loaded_once_and_missing_parts_are_loud(monkeypatch):
    _lib_or_skip()
    assert L.ops() is L.ops() is L.OPS
    for name in L._BOUND:
        assert name in L.SYMBOLS
    import sys
    import rumpy_amd
    monkeypatch.setattr(L, 'OPS', None)
    monkeypatch.delattr(rumpy_amd, '_torch_bind')
    monkeypatch.setitem(sys.modules, 'rumpy_amd._torch_bind', None)         # as if it were not built
    with pytest.raises(RuntimeError, match='no fallback'):
        residual_norm(torch.zeros(2, 8), pre_norm='rms')


def test_contrastive_models_refuse_targets_they_do_not_make():
    from rumpy_amd.regression.models.contrastive_learning.encoding_models import Encoder
    from rumpy_amd.regression.models.contrastive_learning.moco import MoCo
    from rumpy_amd.regression.models.contrastive_learning.supmoco import SupMoCo
    from rumpy_amd.regression.models.contrastive_learning.weak_con import WeakCon
    for kw in ({'distill_top': 0}, {'distill_top': 65}, {'distill_top': 8, 'distill_t': 0.0}, {'distill_top': 8, 'distill_t': float('nan')}):
        with pytest.raises(ValueError, match='distill_t'):
            MoCo(base_encoder=Encoder, K=64, **kw)
    for kind in (SupMoCo, WeakCon):
        with pytest.raises(ValueError, match='%s makes no distillation targets' % kind.__name__):
            kind(device='cpu', base_encoder=Encoder, K=64, distill_top=8)
