"""Layers with 4-bit projections, cache and attention on two streams at once, each with values of its own."""

import pytest
import torch

from mini_hisparse_amd.dense import quantize_weight

from test_four_bit_chain import DIM, HEADS, HIDDEN, KV, Layer


def layer_of(prompts, seed, device):
    """A layer whose every value is drawn from `seed`, after its prompts."""
    layer = Layer(prompts, 30, torch.bfloat16, device)
    layer.gen.manual_seed(seed)

    def draw(*shape):
        return (torch.randn(*shape, generator=layer.gen) * shape[-1] ** -0.5).to(torch.bfloat16).to(device)

    layer.weights = [(torch.rand(DIM, generator=layer.gen) + 0.5).to(torch.bfloat16).to(device) for _ in range(2)]
    layer.into, layer.out = (quantize_weight(draw(n, k)) for n, k in
                             (((HEADS + 2 * KV) * DIM, HIDDEN), (HIDDEN, HEADS * DIM)))
    layer.bias = draw((HEADS + 2 * KV) * DIM)
    for b, n in enumerate(prompts):
        layer.prefill(b, n)
    return layer


@pytest.mark.gpu
@pytest.mark.parametrize("prompts", [[2500, 3, 900], [9000, 40, 7000, 1]])
def test_streams_with_values_of_their_own(gpu, prompts):
    """Parts joined in the launch, and by a second one: what a stream left in the other's workspace would
    show, since no two layers have a value in common."""
    steps, seeds = 10, (1, 2)
    alone, beside = ([layer_of(prompts, seed, gpu) for seed in seeds] for _ in range(2))
    inputs = [[layer.hidden(len(prompts)) for _ in range(steps)] for layer in alone]
    assert not torch.equal(inputs[0][0], inputs[1][0]) and not torch.equal(alone[0].into.tiles, alone[1].into.tiles)
    want = [[layer.decode(x)[1:] for x in xs] for layer, xs in zip(alone, inputs)]
    torch.cuda.synchronize()
    for a, b in zip(*want):  # no request's result is the other layer's
        for x, y in zip(a, b):
            assert (x != y).flatten(1).any(-1).all()
    streams = [torch.cuda.Stream(torch.device(gpu)) for _ in beside]
    got = [[], []]
    for i in range(steps):
        for k, (layer, stream) in enumerate(zip(beside, streams)):
            with torch.cuda.stream(stream):
                got[k].append(layer.decode(inputs[k][i])[1:])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert all(torch.equal(p, q) for p, q in zip(x, y))
