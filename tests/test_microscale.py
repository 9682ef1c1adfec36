"""CPU: the microscaled operators' host side (argument checks of the C ABI and of mapping_challenge_amd.microscale, workspace sizes) and the oracle's own
consistency.  No kernel is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from mapping_challenge_amd import _lib, microscale as mx
from oracle import mx_ref

A16 = 1 << 20        # stands for a device address: the calls below are refused before anything reads it


def refused(rc, *words):
    msg = _lib.load().msc_last_error().decode()
    assert rc < 0, 'accepted'
    for w in words:
        assert w in msg, msg


def test_pack_refusals():
    lib = _lib.load()
    good = dict(x=A16, x_ld=64, dtype=_lib.BF16, codes=A16, codes_ld=64, scales=A16, scales_ld=2, fmt=_lib.MX_E4M3, rows=4, C=64)

    def pack(**kw):
        a = dict(good, **kw)
        return lib.msc_mx_pack(a['x'], a['x_ld'], a['dtype'], a['codes'], a['codes_ld'], a['scales'], a['scales_ld'], a['fmt'], a['rows'], a['C'], None)

    def unpack(**kw):
        a = dict(good, **kw)
        return lib.msc_mx_unpack(a['codes'], a['codes_ld'], a['scales'], a['scales_ld'], a['fmt'], a['x'], a['x_ld'], a['dtype'], a['rows'], a['C'], None)
    for call in (pack, unpack):
        refused(call(fmt=2), 'format')
        refused(call(dtype=3), 'dtype')
        refused(call(rows=-1), 'shape')
        refused(call(C=0), 'shape')
        refused(call(C=(1 << 24) + 1), 'shape')
        refused(call(x=None), 'null')
        refused(call(x_ld=63), 'pitch')
        refused(call(x=A16 + 1), 'aligned')
        refused(call(codes=None), 'codes')
        refused(call(codes=A16 + 8), 'codes')
        refused(call(codes_ld=48), 'codes')
        refused(call(codes_ld=72), 'codes')
        refused(call(scales_ld=1), 'codes')
        refused(call(scales=None), 'codes')
        assert call(rows=0, x=None, codes=None, scales=None) == 0          # nothing to do
    refused(pack(fmt=_lib.MX_E2M1, C=65, x_ld=65, codes_ld=32, scales_ld=3), 'codes')


def wgrad_desc(**kw):
    d = _lib.MxWgradDesc()
    v = dict(p=A16, q=A16, q_scales=A16, dw=A16, ws=A16, p_ld=64, q_ld=64, s_ld=2, dtype=_lib.BF16, N=2, Hp=8, Wp=8, A=64, Hq=8, Wq=8, B=64, KH=3, KW=3, stride=1,
             pad=1)
    for k, x in dict(v, **kw).items():
        setattr(d, k, x)
    return d


def test_weight_gradient_refusals_and_workspace():
    lib = _lib.load()
    run = lambda **kw: lib.msc_mx_wgrad(C.byref(wgrad_desc(**kw)), None)  # noqa: E731
    refused(lib.msc_mx_wgrad(None, None), 'null')
    refused(lib.msc_mx_wgrad_workspace_bytes(None), 'null')
    refused(run(dtype=9), 'dtype')
    for bad in (dict(A=0), dict(B=0), dict(N=-1), dict(Hp=0), dict(Hq=0), dict(A=(1 << 20) + 1)):
        refused(run(**bad), 'shape')
    for bad in (dict(KH=0), dict(KW=17), dict(stride=0), dict(stride=17), dict(pad=-1), dict(pad=17)):
        refused(run(**bad), 'kernel')
    refused(run(N=1 << 20, Hp=64, Wp=64), '2^30')
    refused(run(q_ld=1 << 24), '2^28')
    refused(run(p_ld=1 << 24), '2^24')
    refused(run(N=200, Hp=1, Wp=1, Hq=16, Wq=16, KH=16, KW=16, pad=0, q_ld=1 << 19), '2 GiB')
    for bad in (dict(p=None), dict(dw=None), dict(p_ld=63), dict(p=A16 + 1), dict(dw=A16 + 2)):
        refused(run(**bad), 'tensor')
    for bad in (dict(q=None), dict(q=A16 + 4), dict(q_ld=32), dict(q_ld=68), dict(s_ld=1), dict(q_scales=None)):
        refused(run(**bad), 'E4M3')
    big = dict(N=32, Hp=64, Wp=64, Hq=64, Wq=64)
    assert lib.msc_mx_wgrad_workspace_bytes(C.byref(wgrad_desc(**big))) > 0
    refused(run(ws=None, **big), 'workspace')
    refused(run(ws=A16 + 8, **big), 'workspace')
    assert lib.msc_mx_wgrad_workspace_bytes(C.byref(wgrad_desc(N=1, Hp=1, Wp=5, Hq=1, Wq=5))) == 0      # one range of pixels: no partial sums
    assert lib.msc_mx_wgrad_workspace_bytes(C.byref(wgrad_desc(N=0))) == 0 and run(N=0, accumulate=1) == 0      # no pixels: nothing to add
    refused(run(N=0, dw=None), 'tensor')


def bn_desc(**kw):
    d = _lib.MxBnBwdDesc()
    v = dict(dout=A16, y=A16, y_scales=A16, gamma=A16, mean=A16, invstd=A16, dgamma=A16, dbeta=A16, dy=2 * A16, ws=A16, dout_ld=64, y_ld=64, s_ld=2, dy_ld=64,
             rows=10, dtype=_lib.F16, C=64)
    for k, x in dict(v, **kw).items():
        setattr(d, k, x)
    return d


def test_batchnorm_refusals_and_workspace():
    lib = _lib.load()
    run = lambda **kw: lib.msc_mx_bn_bwd(C.byref(bn_desc(**kw)), None)  # noqa: E731
    refused(lib.msc_mx_bn_bwd(None, None), 'null')
    refused(run(dtype=-1), 'dtype')
    for bad in (dict(rows=0), dict(C=0), dict(rows=-5)):
        refused(run(**bad), 'shape')
        assert lib.msc_mx_bn_bwd_workspace_bytes(bad.get('rows', 1), bad.get('C', 1)) == 0
    for bad in ('dout', 'dy', 'mean', 'invstd', 'ws'):
        refused(run(rows=5000, **{bad: None}), 'null')
    refused(run(relu=1), 'relu')
    refused(run(relu=2), 'scale')
    refused(run(relu=3), 'mask')
    refused(run(relu=3, relu_mask=A16, mask_ld=7), 'mask')
    refused(run(relu=3, relu_mask=A16, mask_ld=8, dtype=_lib.F32), 'mask')
    refused(run(dout_ld=63), 'pitch')
    refused(run(dy_ld=60), 'pitch')
    refused(run(dres=4 * A16, dres_ld=8), 'pitch')
    refused(run(y=A16 + 8), 'E4M3')
    refused(run(ws=A16 + 4), 'workspace')
    refused(run(dout=A16 + 1), 'aligned')
    refused(run(dres=2 * A16, dres_ld=64), 'different')                    # dy and dres in one buffer
    refused(run(dy=A16, dy_ld=80), 'pitch')                                # in place at another pitch
    assert lib.msc_mx_bn_bwd_workspace_bytes(131072, 256) >= 256 * 32 and lib.msc_mx_bn_bwd_workspace_bytes(100, 256) == 0      # few rows: one launch


def linear_desc(**kw):
    d = _lib.MxLinearDesc()
    v = dict(x=A16, w=A16, w_scales=A16, out=2 * A16, ws=A16, x_ld=64, w_ld=32, s_ld=2, out_ld=48, M=5, dtype=_lib.BF16, K=64, N=48)
    for k, x in dict(v, **kw).items():
        setattr(d, k, x)
    return d


def test_linear_refusals_and_workspace():
    lib = _lib.load()
    run = lambda **kw: lib.msc_mx_linear(C.byref(linear_desc(**kw)), None)  # noqa: E731
    refused(lib.msc_mx_linear(None, None), 'null')
    refused(run(dtype=5), 'dtype')
    for bad in (dict(M=-1), dict(K=0), dict(N=0)):
        refused(run(**bad), 'shape')
        assert lib.msc_mx_linear_workspace_bytes(C.byref(linear_desc(**bad))) == -1
    for bad in (dict(out=None), dict(out_ld=47), dict(out=A16 + 1), dict(res=A16, res_ld=40), dict(res=A16 + 1, res_ld=48)):
        refused(run(**bad), 'out')
    refused(run(res=2 * A16, out=2 * A16, res_ld=64, out_ld=48), 'in place')
    refused(run(out=A16, x=A16), 'cannot be x')
    for bad in (dict(w=None), dict(w=A16 + 8), dict(w_ld=16), dict(s_ld=1), dict(w_scales=None)):
        refused(run(**bad), 'E2M1')
    refused(run(x_ld=63), 'x misaligned')
    refused(run(x=A16 + 1), 'x misaligned')
    refused(run(x=None), 'x (or its codes')
    refused(run(x=None, x_codes=A16, x_scales=A16, xc_ld=16, xs_ld=2), 'x (or its codes')
    assert run(M=0) == 0
    many = dict(M=1000, K=4096, N=3000, x_ld=4096, w_ld=2048, s_ld=128, out_ld=3000)      # x is packed by a launch of its own
    assert lib.msc_mx_linear_workspace_bytes(C.byref(linear_desc(**many))) >= 1000 * (2048 + 128)
    refused(run(ws=None, **many), 'workspace')
    refused(run(ws=A16 + 4, **many), 'workspace')
    assert lib.msc_mx_linear_workspace_bytes(C.byref(linear_desc(x=None, **many))) == 0


def test_python_refusals():
    u8 = torch.uint8
    with pytest.raises(ValueError, match='format'):
        mx.MxTensor(torch.zeros(2, 32, dtype=u8), torch.zeros(2, 1, dtype=u8), 32, 'e5m2')
    with pytest.raises(ValueError, match='take 64 code bytes'):
        mx.MxTensor(torch.zeros(2, 32, dtype=u8), torch.zeros(2, 1, dtype=u8), 33)
    with pytest.raises(ValueError, match='uint8'):
        mx.MxTensor(torch.zeros(2, 32), torch.zeros(2, 1, dtype=u8), 32)
    with pytest.raises(ValueError, match='at least one channel'):
        mx.MxTensor(torch.zeros(2, 0, dtype=u8), torch.zeros(2, 0, dtype=u8), 0)
    with pytest.raises(_lib.MscError, match='no CPU path'):
        mx.pack(torch.zeros(2, 32))
    with pytest.raises(ValueError, match='format'):
        mx.pack(torch.zeros(2, 32), 'int8')
    t = mx.empty((2, 40), 'e2m1', 'cpu')
    assert t.shape == (2, 40) and t.nbytes == 2 * (32 + 2) and t.codes.shape == (2, 32)
    with pytest.raises(_lib.MscError, match='no CPU path'):
        mx.unpack(t)
    with pytest.raises(ValueError, match='e4m3'):
        mx.conv_weight_grad(torch.zeros(2, 8), t)
    with pytest.raises(ValueError, match='needs out'):
        mx.conv_weight_grad(torch.zeros(2, 8), mx.empty((2, 40), 'e4m3', 'cpu'), accumulate=True)
    with pytest.raises(ValueError, match='e4m3'):
        mx.batchnorm_backward(torch.zeros(2, 40), t, None, None, None)
    with pytest.raises(ValueError, match='differ'):
        mx.batchnorm_backward(torch.zeros(2, 41), mx.empty((2, 40), 'e4m3', 'cpu'), None, None, None)
    with pytest.raises(ValueError, match='e2m1'):
        mx.linear(torch.zeros(2, 40), mx.empty((8, 40), 'e4m3', 'cpu'))
    with pytest.raises(ValueError, match='go together'):
        mx.linear(torch.zeros(2, 41), mx.empty((8, 40), 'e2m1', 'cpu'))
    with pytest.raises(ValueError, match='type of x'):
        mx.linear(torch.zeros(2, 40), mx.empty((8, 40), 'e2m1', 'cpu'), dtype=torch.float16)


@pytest.mark.parametrize('fmt,half,top', [('e4m3', 2.0 ** -4, 448.0), ('e2m1', 2.0 ** -2, 6.0)])
def test_oracle_packs_to_the_nearest_value(fmt, half, top):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((40, 75)) * np.exp(rng.standard_normal((40, 75)))).astype(np.float32).astype(np.float64)
    x[3] = 0
    codes, scales = mx_ref.pack(x, 'fp32', fmt)
    v = mx_ref.unpack(codes, scales, 75, fmt)
    least = mx_ref.CODES[fmt][1]
    s = np.repeat(np.ldexp(1.0, scales.astype(np.int64) - 127), 32, axis=1)[:, :75]
    assert (np.abs(v - x) <= np.maximum(half * np.abs(x), least / 2 * s)).all()
    assert (np.abs(x) <= top * s).all()                                    # nothing passes the largest code
    amax = np.abs(np.pad(x, ((0, 0), (0, 21)))).reshape(40, 3, 32).max(2)
    assert ((amax > top * np.ldexp(1.0, scales.astype(np.int64) - 128)) | (amax == 0)).all()      # and half the scale would not do
    again, _ = mx_ref.pack(v, 'fp32', fmt)
    assert (mx_ref.unpack(again, _, 75, fmt) == v).all()                   # values are fixed points


def test_oracle_batchnorm_gradient_against_differences():
    rng = np.random.default_rng(5)
    y, gamma, beta, g = rng.standard_normal((7, 3)), rng.standard_normal(3) + 1, rng.standard_normal(3), rng.standard_normal((7, 3))

    def f(y, gamma, beta):
        return (np.maximum(mx_ref.batchnorm_forward(y, gamma, beta, 1e-5)[0], 0) * g).sum()
    out, mean, invstd = mx_ref.batchnorm_forward(y, gamma, beta, 1e-5)
    dy, dgamma, dbeta, _ = mx_ref.batchnorm_backward(g, y, gamma, mean, invstd, out > 0)
    h = 1e-6
    for i in range(7):
        for c in range(3):
            e = np.zeros_like(y)
            e[i, c] = h
            assert abs((f(y + e, gamma, beta) - f(y - e, gamma, beta)) / (2 * h) - dy[i, c]) < 1e-7
    for c in range(3):
        e = np.eye(3)[c] * h
        assert abs((f(y, gamma + e, beta) - f(y, gamma - e, beta)) / (2 * h) - dgamma[c]) < 1e-7
        assert abs((f(y, gamma, beta + e) - f(y, gamma, beta - e)) / (2 * h) - dbeta[c]) < 1e-7


def test_network_option_is_checked():
    from mapping_challenge_amd.unet_models import UNetResNet
    with pytest.raises(ValueError, match='activation_checkpoint'):
        UNetResNet(34, 2, num_filters=32, dropout_2d=0.0, is_deconv=True, activation_checkpoint='int8')
    net = UNetResNet(34, 2, num_filters=32, dropout_2d=0.0, is_deconv=True, activation_checkpoint='e4m3')
    assert net.activation_checkpoint == 'e4m3'
