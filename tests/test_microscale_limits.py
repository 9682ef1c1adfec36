"""CPU: refusals of the microscaled operators at the limits of their arguments.  No kernel is launched."""
import ctypes as C

import pytest
import torch

from mapping_challenge_amd import _lib, microscale as mx
from test_microscale import A16, bn_desc, linear_desc, refused, wgrad_desc


def test_packed_tensor_of_an_unknown_type_is_refused():
    codes, scales = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    assert mx.MxTensor(codes, scales, 40).dtype is None
    assert mx.MxTensor(codes, scales, 40, dtype=torch.bfloat16).dtype == torch.bfloat16
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        mx.MxTensor(codes, scales, 40, dtype=torch.float64)


def test_weight_gradient_sizes_whose_products_pass_64_bits():
    """2^22 * 2^21 * 2^21 pixels are 0 modulo 2^64: the plan divided by it, and the process ended"""
    lib = _lib.load()
    for bad, word in ((dict(N=1 << 22, Hp=1 << 21, Wp=1 << 21), '2^30'), (dict(Hp=1 << 30, Wp=1 << 30), '2^30'), (dict(Hq=1 << 30, Wq=1 << 30, q_ld=32), '2^30'),
                      (dict(Hq=2, Wq=2, q_ld=1 << 62), '2^28'), (dict(Hq=2, Wq=2, s_ld=1 << 62), '2^28'), (dict(Hq=1 << 14, Wq=1 << 14, q_ld=1 << 36), '2^28')):
        assert lib.msc_mx_wgrad_workspace_bytes(C.byref(wgrad_desc(**bad))) == -1
        refused(lib.msc_mx_wgrad(C.byref(wgrad_desc(**bad)), None), word)


def test_batchnorm_of_more_rows_than_any_memory():
    lib = _lib.load()
    for rows in (1 << 40, (1 << 63) - 1):
        assert lib.msc_mx_bn_bwd_workspace_bytes(rows, 64) == 0
        refused(lib.msc_mx_bn_bwd(C.byref(bn_desc(rows=rows)), None), 'shape')
    assert lib.msc_mx_bn_bwd_workspace_bytes((1 << 40) - 1, 64) > 0


def test_linear_refuses_before_it_launches():
    """too many tiles, and rows too far apart for a tile's descriptor: found before x is packed or a row of scales copied (here, without a device, a launch is an error of its own)"""
    lib = _lib.load()
    run = lambda **kw: lib.msc_mx_linear(C.byref(linear_desc(**kw)), None)  # noqa: E731
    refused(run(M=1 << 35, N=2048, out_ld=2048), '2^30')                   # x to be packed
    many = dict(x=None, x_codes=A16, x_scales=A16 + 1, xc_ld=32, xs_ld=3, M=1 << 35, N=2048, out_ld=2048, w_scales=A16 + 1, s_ld=3)
    refused(run(**many), '2^30')                                           # scales to be laid out
    refused(run(M=2000, K=2048, N=3000, out_ld=3000, x_ld=2048, s_ld=64, w_ld=1 << 24), '2 GiB')
    refused(run(M=200, K=2048, N=300, out_ld=300, x_ld=2048, s_ld=64, w_ld=1 << 62), '2 GiB')
    refused(run(M=200, w_ld=1 << 25, N=64, out_ld=64), '2 GiB')            # x quantised by the product's own launch
    far = dict(x=None, x_codes=A16, x_scales=A16, xc_ld=32, xs_ld=2, M=2000, K=2048, N=3000, out_ld=3000, w_ld=1024, s_ld=64, w_scales=A16 + 1)
    refused(run(**dict(far, xc_ld=1 << 24, xs_ld=64)), '2 GiB')
    refused(run(**dict(far, xc_ld=1024, xs_ld=1 << 24)), '2 GiB')
    refused(run(**dict(far, xc_ld=1024, xs_ld=64, w_scales=A16, s_ld=1 << 24)), '2 GiB')


M = 1 << 20        # addresses far from each other


def test_results_that_share_memory_with_operands_are_refused():
    lib = _lib.load()
    pk = lambda x, codes, scales, x_ld=64, c_ld=64, s_ld=2, rows=10: lib.msc_mx_pack(x, x_ld, _lib.BF16, codes, c_ld, scales, s_ld, _lib.MX_E4M3, rows, 64, None)  # noqa: E731
    un = lambda x, codes, scales: lib.msc_mx_unpack(codes, 64, scales, 2, _lib.MX_E4M3, x, 64, _lib.BF16, 10, 64, None)  # noqa: E731
    for call in (pk, un):
        refused(call(M, M, 9 * M), 'shares memory')
        refused(call(M, M + 9 * 128 + 112, 9 * M), 'shares memory')       # the last row's last bytes
        refused(call(M, 9 * M, M + 40), 'shares memory')
    refused(pk(M, M + 32, 9 * M, x_ld=256, c_ld=512), 'shares memory')     # inside the rows' columns

    w = lambda **kw: lib.msc_mx_wgrad(C.byref(wgrad_desc(**dict(dict(p=M, q=4 * M, q_scales=8 * M, dw=12 * M, ws=16 * M), **kw))), None)  # noqa: E731
    for bad in (dict(dw=M), dict(dw=4 * M + 256), dict(dw=8 * M), dict(dw=M - 4), dict(dw=4 * M - 64 * 9 * 64 * 4 + 4)):
        refused(w(**bad), 'shares memory')

    far = dict(dout=M, y=4 * M, y_scales=8 * M, dy=12 * M, dres=16 * M, dres_ld=64, ws=20 * M, relu=3, relu_mask=24 * M, mask_ld=8)
    b = lambda **kw: lib.msc_mx_bn_bwd(C.byref(bn_desc(**dict(far, **kw))), None)  # noqa: E731
    for bad in (dict(dy=M + 128), dict(dy=M - 2), dict(dres=M + 2), dict(dy=4 * M), dict(dres=8 * M), dict(dres=24 * M), dict(dy=16 * M + 64), dict(dy=M + 64, dout_ld=96, dy_ld=96),
                dict(dy=M + 4, dout_ld=256, dy_ld=128)):
        refused(b(**bad), 'memory')

    lin = dict(x=M, w=4 * M, w_scales=8 * M, out=12 * M, res=16 * M, res_ld=48, ws=20 * M)
    n = lambda **kw: lib.msc_mx_linear(C.byref(linear_desc(**dict(lin, **kw))), None)  # noqa: E731
    for bad in (dict(out=M + 2), dict(out=M - 2), dict(out=4 * M), dict(out=8 * M), dict(out=16 * M + 96), dict(out=16 * M - 2), dict(out=M + 126, x_ld=112, out_ld=112),
                dict(x=None, x_codes=24 * M, x_scales=28 * M, xc_ld=32, xs_ld=2, out=24 * M), dict(x=None, x_codes=24 * M, x_scales=28 * M, xc_ld=32, xs_ld=2, out=28 * M)):
        refused(n(**bad), 'memory' if bad.get('out') != 24 * M else 'x')


def test_network_option_set_later_is_checked():
    """the attribute is read when a training program is built: another word would have run as 'e4m3'"""
    from mapping_challenge_amd.unet_models import UNetResNet
    net = UNetResNet(34, 2, num_filters=32, dropout_2d=0.0, is_deconv=True)
    net.activation_checkpoint = 'e5m2'
    with pytest.raises(ValueError, match='activation_checkpoint'):
        net._program(1, 64, 64, True, torch.device('cpu'))
