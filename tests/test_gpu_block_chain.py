"""The block operators together, as one pass of a DiT block uses them: block
selection, attention over the lists, the norms around the branch, the MLP with its
gated activation and gated residual. Each step against 64 bits on the very inputs
that it got; then the pass in a graph, on another stream, and with lists that
change between replays."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import BlockSparseKernel, DenseMiniMaxH3Processor, fused_linear, select_key_blocks, sparse_attn_func
from h3_flash_amd.fusions import fused_rmsnorm_residual_gate_rmsnorm_modulate
from oracle.block import linear_reference, sandwich_reference, select_reference, sparse_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16
H, C, FFN, EPS = 2, 256, 328, 1e-5


class _Block:
    def __init__(self, seed: int) -> None:
        g = torch.Generator(device=DEV).manual_seed(seed)
        randn = lambda *s: torch.randn(s, device=DEV, generator=g)  # noqa: E731
        self.w_in, self.w_out = (randn(2 * FFN, C) * C**-0.5).to(BF16), (randn(C, FFN) * FFN**-0.5).to(BF16)
        self.b_out = (0.1 * randn(C)).to(BF16)
        self.post, self.pre = (1 + 0.1 * randn(C)).to(BF16), (1 + 0.1 * randn(C)).to(BF16)
        self.tables = (0.3 * randn(9, 4 * C)).to(BF16).chunk(4, -1)

    def __call__(self, q, k, v, x, index):
        gate_a, scale, shift, gate_m = self.tables
        lists = select_key_blocks(q, k, 3)
        attn, lse = sparse_attn_func(q, k, v, lists)
        hidden, normed = fused_rmsnorm_residual_gate_rmsnorm_modulate(
            x, attn.flatten(2), self.post, gate_a, self.pre, scale, shift, index, EPS
        )
        act = fused_linear(normed, self.w_in, gated=True, activation="silu")
        out = fused_linear(act, self.w_out, self.b_out, residual=hidden, gate=gate_m, index=index)
        return lists, attn, lse, hidden, normed, act, out


def _inputs(S: int, seed: int):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(s, device=DEV, generator=g).to(BF16)  # noqa: E731
    q, k, v = (randn(1, S, H, 128) for _ in range(3))
    return q, k, v, randn(1, S, C), torch.arange(S, device=DEV) * 9 // S


def _within(got, want, bound):
    worst = ((got.double().cpu().reshape(want.shape) - want.cpu()).abs() / bound.cpu()).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("S", [1, 77, 700])
def test_each_step_of_a_pass(S):
    block = _Block(1)
    q, k, v, x, index = _inputs(S, 2)
    gate_a, scale, shift, gate_m = block.tables
    lists, attn, lse, hidden, normed, act, out = block(q, k, v, x, index)
    assert torch.equal(lists.cpu(), select_reference(q.cpu(), k.cpu(), 3))
    o, ob, l, lb = sparse_reference(q.cpu(), k.cpu(), v.cpu(), lists.cpu())
    _within(attn, o, ob)
    _within(lse, l, lb)
    h, hb, n, nb = sandwich_reference(x, attn.flatten(2), block.post, gate_a, block.pre, scale, shift, index, EPS)
    _within(hidden, h, hb)
    _within(normed, n, nb)
    _within(act, *linear_reference(normed, block.w_in, None, "silu", True))
    _within(out, *linear_reference(act, block.w_out, block.b_out, None, False, hidden, gate_m, index))


@pytest.mark.parametrize("S", [20, 900])
def test_a_pass_in_a_graph(S):
    block = _Block(3)
    static = _inputs(S, 4)
    for _ in range(2):
        block(*static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block(*static)
    for seed in (5, 6, 7):
        fresh = _inputs(S, seed)
        eager = block(*fresh)
        for s, f in zip(static, fresh):
            s.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for c, e in zip(captured, eager):
            assert torch.equal(c, e), (S, seed)


def test_two_graphs_and_eager_calls_share_nothing():
    blocks, inputs = (_Block(8), _Block(9)), (_inputs(300, 10), _inputs(1100, 11))
    want = [b(*i) for b, i in zip(blocks, inputs)]
    torch.cuda.synchronize()
    graphs, captured = [], []
    for b, i in zip(blocks, inputs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            captured.append(b(*i))
    for _ in range(3):
        for g in graphs:
            g.replay()
        again = blocks[0](*inputs[0])
        torch.cuda.synchronize()
        for got, ref in zip((*captured, again), (*want, want[0])):
            for x, y in zip(got, ref):
                assert torch.equal(x, y)


def test_another_stream():
    block, inputs = _Block(12), _inputs(600, 13)
    want = block(*inputs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = block(*inputs)
    stream.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_results_do_not_vary_between_calls():
    block, inputs = _Block(14), _inputs(1300, 15)
    first = block(*inputs)
    for _ in range(5):
        for x, y in zip(block(*inputs), first):
            assert torch.equal(x, y)


def test_processor_takes_the_sparse_kernel():
    class Attention:
        heads, fused_projections = H, False
        norm_q = norm_k = staticmethod(lambda t: t)
        to_out = [torch.nn.Identity(), torch.nn.Identity()]

        def __init__(self):
            g = torch.Generator(device=DEV).manual_seed(16)
            w = [(torch.randn((H * 128, C), device=DEV, generator=g) * C**-0.5).to(BF16) for _ in range(3)]
            self.to_q, self.to_k, self.to_v = ((lambda t, m=m: t @ m.t()) for m in w)

    attn, x = Attention(), _inputs(800, 17)[3]
    kernel = BlockSparseKernel(keep=0.3)
    processor = DenseMiniMaxH3Processor(kernel=kernel)
    got = processor(attn, x)
    q, k, v = (f(x).unflatten(-1, (H, 128)) for f in (attn.to_q, attn.to_k, attn.to_v))
    want = sparse_attn_func(q, k, v, select_key_blocks(q, k, 4))[0].flatten(2)
    assert processor.calls == 1 and torch.equal(got, want)
