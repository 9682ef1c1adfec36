"""GPU: UNetResNet(activation_checkpoint='e4m3') -- the encoder's backward from 8-bit checkpoints -- against the float64 oracle network whose convolutions and
BatchNorms differentiate at inputs that were packed and restored (oracle/mx_ref.py)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import mx_ref, unet_ref

pytestmark = pytest.mark.gpu


def stored(x):
    """NCHW float64 -> what its E4M3 checkpoint holds (the engine in fp32: the values are float32)"""
    r = x.detach().permute(0, 2, 3, 1).contiguous()
    v = mx_ref.unpack(*mx_ref.pack(r.float().double().reshape(-1, r.shape[3]).numpy(), 'fp32', 'e4m3'), r.shape[3], 'e4m3')
    return torch.from_numpy(np.ascontiguousarray(v)).view(r.shape).permute(0, 3, 1, 2).contiguous()


class Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, stride, pad):
        ctx.save_for_backward(stored(x), w)
        ctx.args = stride, pad
        return F.conv2d(x, w, None, stride, pad)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        stride, pad = ctx.args
        return (torch.nn.grad.conv2d_input(x.shape, w, dy, stride, pad), torch.nn.grad.conv2d_weight(x, w.shape, dy, stride, pad), None, None)


class BatchNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, gamma, beta, eps):
        mean, invstd = y.mean((0, 2, 3)), 1 / torch.sqrt(y.var((0, 2, 3), unbiased=False) + eps)
        ctx.save_for_backward(stored(y), gamma, mean, invstd)
        v = lambda t: t.view(1, -1, 1, 1)  # noqa: E731
        return (y - v(mean)) * v(invstd * gamma) + v(beta)

    @staticmethod
    def backward(ctx, g):
        y, gamma, mean, invstd = ctx.saved_tensors
        rows = lambda t: t.permute(0, 2, 3, 1).reshape(-1, t.shape[1]).numpy()  # noqa: E731
        dy, dgamma, dbeta, _ = mx_ref.batchnorm_backward(rows(g), rows(y), gamma.numpy(), mean.numpy(), invstd.numpy())
        n, c, h, w = g.shape
        return torch.from_numpy(dy).view(n, h, w, c).permute(0, 3, 1, 2).contiguous(), torch.from_numpy(dgamma), torch.from_numpy(dbeta), None


def oracle_gradients(depth, sd, x, dout, checkpoints):
    ref = unet_ref.UNetResNetRef(depth)
    ref.load_state_dict(sd)
    ref = ref.double().train()
    if checkpoints:
        for name, m in ref.encoder.named_modules():
            if name in ('conv1', 'bn1'):                                   # the stem stays as it is
                continue
            if isinstance(m, torch.nn.Conv2d):
                m.forward = lambda t, m=m: Conv.apply(t, m.weight, m.stride[0], m.padding[0])
            elif isinstance(m, torch.nn.BatchNorm2d):
                m.forward = lambda t, m=m: BatchNorm.apply(t, m.weight, m.bias, m.eps)
    ref(x.double()).backward(dout.double())
    return {n: p.grad for n, p in ref.named_parameters() if p.grad is not None}


def network(depth, sd, dtype, checkpoint):
    from mapping_challenge_amd.unet_models import UNetResNet
    net = UNetResNet(depth, 2, num_filters=32, dropout_2d=0.0, is_deconv=True, compute_dtype=dtype, autotune=False, activation_checkpoint=checkpoint)
    net.load_state_dict(sd)
    net.flatten_parameters('cuda')
    return net.train()


def engine_gradients(net, x, dout):
    net.zero_grad()
    net(x.cuda()).backward(dout.cuda())
    return {n: p.grad.detach().double().cpu() for n, p in net.named_parameters() if p.grad is not None}


def distances(a, b):
    return np.array([float((a[n] - b[n]).norm() / b[n].norm()) for n in b if n in a and b[n].norm() > 0])


@pytest.mark.parametrize('depth', [34, 101])
def test_gradients_from_checkpoints(depth):
    """fp32 engine: its gradients are the oracle's with packed inputs.  Both compute in higher precision than the checkpoints hold, so what is left between them is fp32
    rounding, and a code here and there where it tips a value over the middle between two: an element then moves by a whole step (2^-3) instead of half, one in thousands"""
    sd = unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(depth))
    x = unet_ref.synthetic_batch(2, 64, 64)
    dout = torch.randn((2, 2, 64, 64), generator=torch.Generator().manual_seed(3)) * 1e-2
    want, plain = oracle_gradients(depth, sd, x, dout, True), oracle_gradients(depth, sd, x, dout, False)
    net = network(depth, sd, 'fp32', 'e4m3')
    got = engine_gradients(net, x, dout)
    near, far = distances(got, want), distances(got, plain)
    print('to the oracle with checkpoints: median %.2e worst %.2e; without: median %.2e worst %.2e' % (np.median(near), near.max(), np.median(far), far.max()))
    assert np.median(near) < 0.1 * np.median(far) and near.max() < far.max()
    assert np.median(far) < 2.0 ** -3                                      # rounding to 3 bits: each factor off by 2^-4 at most
    again = engine_gradients(net, x, dout)                                 # a second step over the same buffers
    assert np.median(distances(again, got)) < 1e-3


@pytest.mark.parametrize('depth,dtype', [(34, 'bf16'), (101, 'bf16'), (34, 'fp16')])
def test_forward_is_unchanged(depth, dtype):
    sd = unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(depth))
    x = unet_ref.synthetic_batch(4, 128, 128).cuda()
    a, b = network(depth, sd, dtype, None), network(depth, sd, dtype, 'e4m3')
    pa, pb = a.train_forward(x), b.train_forward(x)
    # the same kernels on the same numbers; the batch statistics are summed by atomics in any order
    scale = pa.logits.abs().max()
    assert (pa.logits - pb.logits).abs().max() <= scale * (2e-2 if dtype == 'bf16' else 4e-3)
    enc = sum(1 for fn, _ in pb.bwd if fn.__name__ == 'msc_mx_wgrad')
    assert enc == sum(1 for n, m in b.encoder.named_modules() if isinstance(m, torch.nn.Conv2d)) - 1


def test_memory_of_a_training_program():
    """ResNet101, batch 8, 256 x 256.  A block of width p keeps 12 p elements per pixel (three raw outputs, three activations: 24 p bytes) and the activations' gradients (12 p
    bytes); with checkpoints 12 p codes, their scales and 6 p mask bits: 13.1 p of 36 p bytes.  Over the stages (pixels x p: 2.1, 1.0, 0.52, 0.26 million, 3 + 4 +
    23 + 3 blocks) that is 840 -> 306 MB, and 55 MB of shared buffers, out of some 1380 MB with the stem, the skips and the decoder"""
    sd = unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(101))
    sizes = {}
    for c in (None, 'e4m3'):
        net = network(101, sd, 'bf16', c)
        p = net.train_forward(unet_ref.synthetic_batch(8, 256, 256).cuda())
        sizes[c] = p.bytes
        del net, p
    print('buffers %.0f MB -> %.0f MB' % (sizes[None] / 1e6, sizes['e4m3'] / 1e6))
    assert sizes['e4m3'] < sizes[None] - 0.9 * (840e6 - 306e6 - 55e6) + 40e6      # up to 34 MB of scratch for partial weight gradients


def test_train_step_with_checkpoints_in_a_graph():
    """TrainStep over the checkpointed network: captured, replayed, the parameters near those of the eager steps"""
    from mapping_challenge_amd.trainer import HipAdam, LossSpec, TrainStep
    from oracle import losses_ref
    sd = unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(34))
    x, t = unet_ref.synthetic_batch(2, 64, 64).cuda(), losses_ref.synthetic_target(2, 64, 64)[:, :1].contiguous().cuda()
    out = []
    for graph in (False, True):
        net = network(34, sd, 'fp32', 'e4m3')
        step = TrainStep(net, LossSpec.plain_ce(), HipAdam(net, lr=1e-4), use_graph=graph)
        losses = []
        for _ in range(4):
            losses.append(step(x, t).item())
            torch.cuda.synchronize()
        assert np.isfinite(losses).all() and (step.graph is not None) == graph
        out.append((losses, net.flat_params.clone(), net.flat_grads.clone()))
    (la, pa, _), (lb, pb, _) = out
    assert np.allclose(la, lb, rtol=1e-3)
    assert float((pa - pb).norm() / pa.norm()) < 1e-4


def test_transformer_takes_the_option():
    from mapping_challenge_amd import models
    arch = {'model_params': {'encoder': 'ResNet34', 'compute_dtype': 'bf16'}, 'optimizer_params': {'lr': 1e-4}, 'regularizer_params': {}}
    train = {'epochs': 1, 'activation_checkpoint': 'e4m3'}
    try:
        t = models.PyTorchUNet(arch, train, {})
    except KeyError as e:
        pytest.skip('configuration key %s' % e)
    assert t.model.activation_checkpoint == 'e4m3'
    with pytest.raises(ValueError, match='activation_checkpoint'):
        models.PyTorchUNet(arch, dict(train, activation_checkpoint='fp8'), {})


@pytest.mark.parametrize('depth', [34, 101])
def test_pieces_of_the_backward_leave_final_gradients(depth):
    """the data-parallel step sends a range of the gradients off as soon as the launches in front of a cut are enqueued: nothing behind the cut may write it again"""
    from mapping_challenge_amd.trainer import ddp_plan
    from mapping_challenge_amd.unet_models import _Program
    net = network(depth, unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(depth)), 'bf16', 'e4m3')
    x = unet_ref.synthetic_batch(2, 64, 64).cuda()
    prog = net.train_forward(x)
    prog.dlogits.copy_(torch.randn(prog.dlogits.shape, generator=torch.Generator().manual_seed(3)) * 1e-2)
    flat = net.flat_grads
    plan, kept, beg = ddp_plan(prog, flat, nchunks=4), [], 0
    assert len(plan) == 4 and sum(hi - lo for _, lo, hi in plan if lo is not None) == flat.numel()
    assert sum(lo is not None for _, lo, _ in plan) >= 3                   # the encoder's gradients leave in pieces too
    flat.zero_()
    prog.stem_dw.zero_()
    for end, lo, hi in plan:
        _Program.run_backward(prog.bwd[beg:end], flat.device)
        beg = end
        if lo is not None:
            kept.append((lo, hi, flat[lo:hi].clone()))
    for lo, hi, then in kept:
        assert torch.equal(flat[lo:hi], then) and torch.isfinite(then).all()
