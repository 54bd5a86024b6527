"""The operators of a decode step in 4 bits as they are used together: 4-bit projections, normed rotary
embedding into a 4-bit cache, attention over it whole and through a window; eager, and captured
once and replayed."""

import pytest
import torch

from mini_hisparse_amd.dense import linear_quantized, norm_rotary_append, quantize_weight
from mini_hisparse_amd.quantized import QuantizedPool
from mini_hisparse_amd.row_kernels import attend_pages

from page_cases import FP4, check as check_attention
from test_linear_quantized import check as check_linear, unpack
from test_norm_rotary import check as check_norm, formula as norm_formula
from test_rotary_append import check_keys, planes

HEADS, KV, DIM, PAGE, EPS, THETA = 14, 2, 64, 16, 1e-6, 1e6
WINDOW, SINKS, HIDDEN = 40, 4, 288


class Batch:
    """Requests of one layer over a paged 4-bit pool: tables, lengths and what a step reads."""

    def __init__(self, prompts, room, dtype, device, seed=0):
        gen = torch.Generator().manual_seed(seed)
        pages = [-(-(n + room) // PAGE) for n in prompts]
        blocks = sum(pages) + 2
        order = torch.randperm(blocks, generator=gen).to(torch.int32)
        self.tables = torch.full((len(prompts), max(pages)), -1, dtype=torch.int32)
        first = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = order[first : first + n]
            first += n
        self.tables = self.tables.to(device)
        self.lengths = torch.zeros(len(prompts), dtype=torch.int32, device=device)
        self.pool = QuantizedPool.empty(blocks, PAGE, KV, DIM, FP4, device)
        self.weights = [(torch.rand(DIM, generator=gen) + 0.5).to(dtype).to(device) for _ in range(2)]
        self.gen, self.dtype, self.device = gen, dtype, device

    def projection(self, rows):
        return (torch.randn(rows, (HEADS + 2 * KV) * DIM, generator=self.gen) * 2).to(self.dtype).to(self.device)

    def prefill(self, request, tokens):
        positions = torch.arange(tokens, device=self.device)
        rows = self.tables[request].long()[positions // PAGE] * PAGE + positions % PAGE
        qkv = self.projection(tokens)
        q = norm_rotary_append(qkv, *self.weights, EPS, positions, rows, self.pool, HEADS, THETA)
        self.lengths[request] = tokens
        return qkv, q, positions, rows

    def step(self, qkv):
        """One new token of every request, with no host value in it: capturable."""
        positions = self.lengths.long()
        rows = self.tables.long().gather(1, (positions // PAGE)[:, None])[:, 0] * PAGE + positions % PAGE
        q = norm_rotary_append(qkv, *self.weights, EPS, positions, rows, self.pool, HEADS, THETA)
        self.lengths += 1
        whole = attend_pages(q, self.pool, self.tables, self.lengths)
        near = attend_pages(q, self.pool, self.tables, self.lengths, window=WINDOW, sinks=SINKS)
        return q, rows, positions, whole, near

    def check(self, qkv, q, positions, rows):
        (want_q, want_k), (size_q, size_k), _ = norm_formula(qkv, *self.weights, EPS, positions, HEADS, KV, DIM, THETA)
        check_norm(q, want_q, size_q, self.dtype)
        got, scales = planes(self.pool)
        check_keys(got[0, rows.cpu()], scales[0, rows.cpu()], want_k, size_k, FP4, self.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prompts_then_decode_steps(gpu, dtype):
    prompts = [70, 1, 33]
    batch = Batch(prompts, 6, dtype, gpu)
    for b, n in enumerate(prompts):
        batch.check(*batch.prefill(b, n))
    for _ in range(5):
        qkv = batch.projection(3)
        q, rows, positions, whole, near = batch.step(qkv)
        batch.check(qkv, q, positions, rows)
        args = (q, batch.pool, batch.tables, batch.lengths)
        check_attention(whole, args)
        check_attention(near, args, WINDOW, SINKS)


@pytest.mark.gpu
@pytest.mark.parametrize("prompts", [[70, 1, 33], [5000, 2, 1900, 700]])
def test_captured_steps(gpu, prompts):
    """The step captured once: every replay writes the next rows and attends over them as the
    eager step does, over page borders, with eager work between the replays."""
    batches = [Batch(prompts, 40, torch.bfloat16, gpu) for _ in range(2)]
    for batch in batches:
        for b, n in enumerate(prompts):
            batch.prefill(b, n)
    eager, captured = batches
    qkv = captured.projection(len(prompts))
    eager.projection(len(prompts))  # keeps the generators alike
    kept, lengths = planes(captured.pool), captured.lengths.clone()
    side = torch.cuda.Stream(torch.device(gpu))
    side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
    with torch.cuda.stream(side):  # a call outside the graph first, its length undone
        captured.step(qkv)
        captured.lengths.copy_(lengths)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, _, _, whole, near = captured.step(qkv)
    for _ in range(20):
        fresh = captured.projection(len(prompts))
        assert torch.equal(fresh, eager.projection(len(prompts)))
        _, _, _, want_whole, want_near = eager.step(fresh)
        qkv.copy_(fresh)
        graph.replay()
        assert torch.equal(whole, want_whole) and torch.equal(near, want_near)
        assert torch.equal(captured.lengths, eager.lengths)
        for x, y in zip(planes(captured.pool), planes(eager.pool)):
            assert torch.equal(x, y)
    assert not torch.equal(planes(captured.pool)[0], kept[0])


class Layer(Batch):
    """A layer's attention with 4-bit projections around it."""

    def __init__(self, prompts, room, dtype, device):
        super().__init__(prompts, room, dtype, device)
        draw = lambda *shape: (torch.randn(*shape, generator=self.gen) * shape[-1] ** -0.5).to(dtype).to(device)  # noqa: E731
        self.into, self.out = (quantize_weight(draw(n, k)) for n, k in
                               (((HEADS + 2 * KV) * DIM, HIDDEN), (HIDDEN, HEADS * DIM)))
        self.bias = draw((HEADS + 2 * KV) * DIM)

    def hidden(self, rows):
        return torch.randn(rows, HIDDEN, generator=self.gen).to(self.dtype).to(self.device)

    def decode(self, x):
        qkv = linear_quantized(x, self.into, self.bias)
        near = self.step(qkv)[-1]
        return qkv, near, linear_quantized(near.flatten(1), self.out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_layer_with_its_projections(gpu, dtype):
    """Each projection is its product's, and the captured layer follows the eager one."""
    prompts = [200, 1, 33, 64]
    eager, captured = (Layer(prompts, 30, dtype, gpu) for _ in range(2))
    for layer in (eager, captured):
        for b, n in enumerate(prompts):
            layer.prefill(b, n)
    x = captured.hidden(len(prompts))
    eager.hidden(len(prompts))
    lengths = captured.lengths.clone()
    captured.decode(x)  # outside the graph first, its length undone
    captured.lengths.copy_(lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = captured.decode(x)[-1]
    for _ in range(12):
        fresh = captured.hidden(len(prompts))
        assert torch.equal(fresh, eager.hidden(len(prompts)))
        qkv, near, want = eager.decode(fresh)
        check_linear(qkv, fresh, *unpack(eager.into), eager.bias)
        check_linear(want, near.flatten(1), *unpack(eager.out), None)
        x.copy_(fresh)
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Layers of their own on two streams, launched in turn with no wait between them, give what each
    gives alone (parts joined in the launch, and by a second one)."""
    for prompts in ([2500, 3, 900], [9000, 40, 7000, 1]):
        alone, beside = ([Layer(prompts, 30, torch.bfloat16, gpu) for _ in range(2)] for _ in range(2))
        inputs = []
        for pair in (alone, beside):
            for layer in pair:
                for b, n in enumerate(prompts):
                    layer.prefill(b, n)
        for layer in alone:
            inputs.append([layer.hidden(len(prompts)) for _ in range(10)])
        want = [[layer.decode(x)[-1] for x in xs] for layer, xs in zip(alone, inputs)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(torch.device(gpu)) for _ in beside]
        got = [[], []]
        for i in range(10):
            for k, (layer, stream) in enumerate(zip(beside, streams)):
                with torch.cuda.stream(stream):
                    got[k].append(layer.decode(inputs[k][i])[-1])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
