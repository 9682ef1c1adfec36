"""GPU: UNetResNet(activation_checkpoint='e4m3') where its layers take the forms of a real step, in the 16-bit engines, and next to the same network without checkpoints."""
import numpy as np
import pytest
import torch

from oracle import unet_ref
from test_gpu_checkpoints import distances, engine_gradients, network, oracle_gradients

pytestmark = pytest.mark.gpu


def case(depth, n, size):
    sd = unet_ref.seeded_state_dict(unet_ref.UNetResNetRef(depth))
    return sd, unet_ref.synthetic_batch(n, size, size), torch.randn((n, 2, size, size), generator=torch.Generator().manual_seed(3)) * 1e-2


@pytest.mark.parametrize('depth,n,size', [(34, 2, 192), (101, 4, 128)])
def test_gradients_of_more_than_2048_rows(depth, n, size):
    """The first stage has 4608 (4096) rows: its BatchNorms go by three launches.  Of the fp32 engine's distance to the network with packed inputs, one part is what the engine without
    checkpoints is away from its own oracle (here a few 1e-3: fp32 through that many layers), the other the elements that such a difference tips into the next code.  One in a
    thousand of them, off by a step where the rest is off by step / sqrt(12) at random, is sqrt(12e-3) = 0.11 of the checkpoints' own effect."""
    sd, x, dout = case(depth, n, size)
    want, plain = oracle_gradients(depth, sd, x, dout, True), oracle_gradients(depth, sd, x, dout, False)
    near = distances(engine_gradients(network(depth, sd, 'fp32', 'e4m3'), x, dout), want)
    own = distances(engine_gradients(network(depth, sd, 'fp32', None), x, dout), plain)
    effect = distances(want, plain)
    print('to the oracle with checkpoints: median %.2e worst %.2e; without, both: %.2e %.2e; the oracles: %.2e %.2e'
          % (np.median(near), near.max(), np.median(own), own.max(), np.median(effect), effect.max()))
    assert np.median(near) <= np.median(own) + 0.11 * np.median(effect)
    assert near.max() <= own.max() + 0.5 * effect.max()                    # the worst layer too: a stage that goes wrong by itself shows here


@pytest.mark.parametrize('depth,dtype', [(34, 'bf16'), (34, 'fp16'), (101, 'bf16')])
def test_gradients_of_the_16_bit_engines(depth, dtype):
    """The forward is the same bits with and without checkpoints, so the gradients differ by what packing rounds: each input by 2^-4 of it at most, 2^-4 / sqrt(3) in the middle
    of its errors, and twice on a gradient's way (the convolution's input, and the BatchNorm's in the gradient that reaches it)."""
    sd, x, dout = case(depth, 2, 64)
    a = engine_gradients(network(depth, sd, dtype, 'e4m3'), x, dout)
    b = engine_gradients(network(depth, sd, dtype, None), x, dout)
    d = distances(a, b)
    print('%s: median %.2e worst %.2e' % (dtype, np.median(d), d.max()))
    assert np.isfinite(d).all() and np.median(d) <= 2.0 ** -4 * np.sqrt(2 / 3) and d.max() <= 2.0 ** -3
    assert np.median(d) > 2.0 ** -8                                        # and packing does happen


@pytest.mark.parametrize('depth,dtype,near', [(34, 'fp32', 2.0 ** -18), (101, 'fp32', 2.0 ** -18), (101, 'bf16', 2.0 ** -8), (34, 'fp16', 2.0 ** -10)])
def test_activations_are_unchanged(depth, dtype, near):
    """Every stage's output and the logits of the training forward, with checkpoints and without, within a rounding of the type on average (in float32 a few).  The same kernels on the same
    numbers: what could differ is the last bit of a batch statistic, summed in double by atomics in any order.  An activation that had been packed would be 2^-5 away."""
    sd, x, _ = case(depth, 4, 128)
    acts = []
    for checkpoint in (None, 'e4m3'):
        p = network(depth, sd, dtype, checkpoint).train_forward(x.cuda())
        acts.append({k: v.float().clone() for k, v in list(p.acts.items()) + [('logits', p.logits)] if v is not None and (k.startswith('cat') or k == 'logits')})
    assert sorted(acts[0]) == ['cat2', 'cat3', 'cat4', 'cat5', 'logits']
    for k, a in acts[0].items():
        assert float((acts[1][k] - a).norm()) <= near * float(a.norm()), k


def test_transformers_hand_the_option_to_the_network():
    from mapping_challenge_amd import models
    arch = {'model_params': {'encoder': 'ResNet34', 'compute_dtype': 'bf16'}, 'optimizer_params': {'lr': 1e-4}, 'regularizer_params': {}}
    assert models.PyTorchUNet(arch, {'epochs': 1, 'activation_checkpoint': 'e4m3'}, {}).model.activation_checkpoint == 'e4m3'
    assert models.PyTorchUNet(arch, {'epochs': 1}, {}).model.activation_checkpoint is None
