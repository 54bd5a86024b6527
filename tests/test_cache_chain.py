"""The cache operators as a decode step uses them: normed rotary split of the projection,
quantised append, attention over page tables; eager, and captured once and replayed."""

import pytest
import torch

from mini_hisparse_amd.dense import norm_rotary_split
from mini_hisparse_amd.quantized import QuantizedPool, append_quantized, read_quantized
from mini_hisparse_amd.row_kernels import attend_pages
from mini_hisparse_amd.selection import quest_topk

from test_attend_pages import check as check_attention
from test_norm_rotary import check as check_norm, formula as norm_formula
from test_quantized import check_append, copy_of

HEADS, KV, DIM, PAGE, EPS, THETA = 14, 2, 64, 16, 1e-6, 1e6


class Batch:
    """Requests of one layer over a paged 8-bit pool: tables, lengths and what a step reads."""

    def __init__(self, prompts, room, code, dtype, device, seed=0):
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
        self.pool = QuantizedPool.empty(blocks, PAGE, KV, DIM, code, device)
        width = (HEADS + 2 * KV) * DIM
        self.weights = [(torch.rand(DIM, generator=gen) + 0.5).to(dtype).to(device) for _ in range(2)]
        self.gen, self.width, self.dtype, self.device = gen, width, dtype, device

    def projection(self, rows):
        return (torch.randn(rows, self.width, generator=self.gen) * 2).to(self.dtype).to(self.device)

    def rows_at(self, request, positions):
        """Physical rows of a request's token positions."""
        return self.tables[request].long()[positions // PAGE] * PAGE + positions % PAGE

    def split(self, qkv, positions):
        return norm_rotary_split(qkv, *self.weights, EPS, positions, HEADS, KV, DIM, THETA)

    def prefill(self, request, tokens):
        """A prompt's rows written in one call; returns its K and V as the cache holds them."""
        positions = torch.arange(tokens, device=self.device)
        _, k, v = self.split(self.projection(tokens), positions)
        rows = self.rows_at(request, positions)
        append_quantized(k, v, rows, self.pool)
        self.lengths[request] = tokens
        return k, v, read_quantized(self.pool, rows, self.dtype)

    def step(self, qkv):
        """One new token of every request, with no host value in it: capturable."""
        positions = self.lengths.long()
        q, k, v = self.split(qkv, positions)
        rows = self.tables.long().gather(1, (positions // PAGE)[:, None])[:, 0] * PAGE + positions % PAGE
        append_quantized(k, v, rows, self.pool)
        self.lengths += 1
        return q, k, v, rows, attend_pages(q, self.pool, self.tables, self.lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prompts_then_decode_steps(gpu, code, dtype):
    prompts = [70, 1, 33]
    batch = Batch(prompts, 6, code, dtype, gpu)
    for b, n in enumerate(prompts):
        k, v, back = batch.prefill(b, n)
        for x, y in zip((k, v), back):
            # the code is within half a step of the quotient (int8: 1/2; e4m3: half of 2^5 at the top
            # of the range), and the value read is rounded to the dtype and, before that, to fp32
            largest = x.float().abs().amax(-1, keepdim=True).double()
            step = 0.5 / 127 if code == torch.int8 else 16.0 / 448
            tol = largest * step * (1 + 2.0**-20) + x.double().abs() * (torch.finfo(dtype).eps + 2.0**-20)
            assert ((x.double() - y.double()).abs() <= tol).all()
    for _ in range(5):
        qkv, before, positions = batch.projection(3), copy_of(batch.pool), batch.lengths.long()
        q, k, v, rows, out = batch.step(qkv)
        (want_q, want_k), (size_q, size_k), want_v = norm_formula(qkv, *batch.weights, EPS, positions, HEADS, KV, DIM,
                                                                  THETA)
        check_norm(q, want_q, size_q, dtype)
        check_norm(k, want_k, size_k, dtype)
        assert torch.equal(v.double().cpu(), want_v)
        check_append(k, v, rows, batch.pool, before)
        check_attention(out, (q, batch.pool, batch.tables, batch.lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("prompts", [[70, 1, 33], [5000, 2, 1900, 700]])
def test_captured_steps(gpu, prompts):
    """The step captured once: every replay writes the next rows and attends over them as the
    eager step does, over page borders, with eager work between the replays."""
    batches = [Batch(prompts, 40, torch.int8, torch.bfloat16, gpu) for _ in range(2)]
    for batch in batches:
        for b, n in enumerate(prompts):
            batch.prefill(b, n)
    eager, captured = batches
    qkv = captured.projection(len(prompts))
    eager.projection(len(prompts))  # keeps the generators alike
    side = torch.cuda.Stream(torch.device(gpu))
    with torch.cuda.stream(side):  # a call outside the graph first, undone
        kept = copy_of(captured.pool)
        lengths = captured.lengths.clone()
        captured.step(qkv)
        captured.lengths.copy_(lengths)
        captured.pool.codes.copy_(kept.codes)
        captured.pool.scales.copy_(kept.scales)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step(qkv)[-1]
    for _ in range(20):
        fresh = captured.projection(len(prompts))
        assert torch.equal(fresh, eager.projection(len(prompts)))
        want = eager.step(fresh)[-1]
        qkv.copy_(fresh)
        graph.replay()
        assert torch.equal(out, want)
        assert torch.equal(captured.pool.codes, eager.pool.codes)
        assert torch.equal(captured.pool.scales, eager.pool.scales)
        assert torch.equal(captured.lengths, eager.lengths)


@pytest.mark.gpu
def test_pages_selected_for_each_kv_head(gpu):
    """Quest pages of each KV head (bounds of the keys as written) attended by tables of its own."""
    tokens, top = 16 * 40 + 5, 8
    batch = Batch([tokens], 1, torch.float8_e4m3fn, torch.bfloat16, gpu)
    k, _, _ = batch.prefill(0, tokens)
    pages = -(-tokens // PAGE)
    padded = torch.cat((k, k[-1:].expand(pages * PAGE - tokens, -1, -1))).view(pages, PAGE, KV, DIM)
    low, high = padded.amin(1).contiguous(), padded.amax(1).contiguous()
    query = batch.split(batch.projection(1), batch.lengths.long())[0]
    leaders = query.view(1, KV, HEADS // KV, DIM)[:, :, 0].contiguous()  # one query of each group chooses
    chosen = quest_topk(leaders, [low], [high], [tokens], PAGE, top)  # [1, KV, top] ascending, the tail last
    tables = batch.tables[0][chosen.long()]
    lengths = torch.tensor([(top - 1) * PAGE + tokens - (pages - 1) * PAGE], dtype=torch.int32, device=gpu)
    args = (query, batch.pool, tables, lengths)
    check_attention(attend_pages(*args), args)
