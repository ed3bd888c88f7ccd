"""The 8-bit operators together, as a block runs them: norm, gated up projection and
down projection without a bf16 tensor between them; captured, replayed, on other streams
and over more than 2^31 values."""

from __future__ import annotations

import ctypes

import pytest
import torch

from h3_flash_amd import _ext, fused_linear, fused_linear_fp8, quantize_fp8, quantize_fp8_weight
from h3_flash_amd.fusions import fused_residual_gate_rmsnorm_modulate, fused_residual_gate_rmsnorm_modulate_fp8, fused_rmsnorm_modulate_fp8
from oracle.fp8 import dequantized
from test_gpu_fp8 import BF16, DEV, _activations, _check, _randn, _same

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Block:
    """The MLP half of a block: weights in bf16 and, quantised once, in 8 bits."""

    def __init__(self, width: int, inner: int, seed: int = 0) -> None:
        self.up = _randn(2 * inner, width, seed=seed + 1, scale=width**-0.5)
        self.down = _randn(width, inner, seed=seed + 2, scale=inner**-0.5)
        self.up8, self.down8 = quantize_fp8_weight(self.up, gated=True), quantize_fp8_weight(self.down)
        self.norm = 1 + _randn(width, seed=seed + 3, scale=0.1)
        self.tables = _randn(5, 4 * width, seed=seed + 4, scale=0.3).chunk(4, -1)
        self.bias = _randn(width, seed=seed + 5, scale=0.1)

    def run8(self, residual, branch, index):
        gate, scale, shift, gate2 = self.tables
        hidden, q, s = fused_residual_gate_rmsnorm_modulate_fp8(residual, branch, gate, self.norm, scale, shift, index, EPS)
        h, hs = fused_linear_fp8(q, *self.up8, x_scale=s, activation="silu", gated=True, quantize=True)
        return (hidden, q, s, h, hs, fused_linear_fp8(h, *self.down8, self.bias, x_scale=hs, residual=hidden, gate=gate2, index=index))

    def run16(self, residual, branch, index):
        gate, scale, shift, gate2 = self.tables
        hidden, n = fused_residual_gate_rmsnorm_modulate(residual, branch, gate, self.norm, scale, shift, index, EPS)
        h = fused_linear(n, self.up, activation="silu", gated=True)
        return hidden, h, fused_linear(h, self.down, self.bias, residual=hidden, gate=gate2, index=index)


def _inputs(m, width, seed=0):
    return _randn(m, width, seed=seed + 7, scale=2.0), _activations(m, width, seed + 8), torch.arange(m, device=DEV) * 5 // m


@pytest.mark.parametrize("m", [1, 20, 33, 390, 1297])
def test_mlp_of_a_block(m):
    width, inner = 1040, 2832
    block = Block(width, inner)
    residual, branch, index = _inputs(m, width)
    hidden, q, s, h, hs, y = block.run8(residual, branch, index)
    # each product on the operands that the step before it left
    _check((h, hs), True, q, s, *block.up8, None, activation="silu", gated=True)
    _check(y, False, h, hs, *block.down8, block.bias, residual=hidden, gate=block.tables[3], index=index)
    # and as a whole, next to bf16: the same hidden state, and the rest off by what the
    # roundings to 8 bits make of it. One rounding has half a step of 2^-4 / mantissa of
    # the value, uniform: 2^-4 / sqrt(6) of a vector's norm (1 / 3 of the square, times
    # the mean of 1 / mantissa^2, a half). h has seen five that count (both operands of
    # its value and of its gate, and its own: sqrt(5) < 3), the branch one more
    # (sqrt(6) < 4); bf16's are 2^-4 of these.
    hidden16, h16, y16 = block.run16(residual, branch, index)
    assert torch.equal(hidden, hidden16)
    step = 2.0**-4 / 6**0.5
    off = (dequantized(h, hs) - h16.double()).norm() / h16.double().norm()
    assert off < 3 * step, off
    branch8, branch16 = y.double() - hidden.double(), y16.double() - hidden.double()
    off = (branch8 - branch16).norm() / branch16.norm()
    assert off < 4 * step, off


def test_attention_output_through_its_projection():
    heads = _randn(1, 390, 8, 128, seed=3)  # (batch, tokens, heads, 128)
    w = _randn(1040, 1024, seed=4, scale=1 / 32)
    wq, ws = quantize_fp8_weight(w)
    q, s = quantize_fp8(heads.flatten(2))
    assert q.shape == (1, 390, 1024) and s.shape == (1, 390, 8)
    y = fused_linear_fp8(q, wq, ws, x_scale=s)
    _check(y, False, q, s, wq, ws, None)
    assert torch.equal(y, fused_linear_fp8(heads.flatten(2), wq, ws))


@pytest.mark.parametrize("m", [9, 300])
def test_captured_and_replayed(m):
    width, inner = 1040, 1296
    block = Block(width, inner)
    residual, branch, index = _inputs(m, width)
    want = [t.clone() for t in block.run8(residual, branch, index)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block.run8(residual, branch, index)
        from_bf16 = fused_linear_fp8(branch, *block.up8, gated=True, activation="gelu")
    for i in range(4):
        fresh, more, _ = _inputs(m, width, seed=10 * i)
        residual.copy_(fresh)
        branch.copy_(more)
        graph.replay()
        eager = block.run8(residual, branch, index)  # the program's own work between replays
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        assert torch.equal(from_bf16, fused_linear_fp8(branch, *block.up8, gated=True, activation="gelu"))
        if i == 0:
            for a, b in zip(got, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_graphs_of_one_pool_and_two_streams():
    # pieces along k and rows rounded first: both take a workspace
    m, k, n = 200, 8208, 1032
    w = quantize_fp8_weight(_randn(n, k, seed=1, scale=0.01))
    xs = [_activations(m, k, s) for s in (1, 2)]
    want = [fused_linear_fp8(x, *w) for x in xs]
    pool, graphs, got = torch.cuda.graph_pool_handle(), [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            got.append(fused_linear_fp8(x, *w))
        graphs.append(graph)
    for _ in range(3):
        for graph, y, ref in zip(graphs, got, want):
            graph.replay()
            assert torch.equal(y, ref)
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(fused_linear_fp8(xs[i], *w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in outs[i])


@pytest.mark.parametrize("x8", [False, True])
def test_the_c_call_with_less_than_the_whole_workspace(x8):
    # pieces along k where it fits, whole tiles where it does not, nothing behind it written
    m, k, n = 200, 8208, 1032
    x, (w, ws) = _activations(m, k, 1), quantize_fp8_weight(_randn(n, k, seed=2, scale=0.01))
    q, s = quantize_fp8(x)
    lib = _ext.load_library()
    for short in (False, True):
        y = torch.full((m + 3, n), 7.0, dtype=BF16, device=DEV)
        of_x = dict(x=q.data_ptr(), x_dtype=4, x_scale=s.data_ptr(), x_scale_stride=s.stride(0)) if x8 else dict(x=x.data_ptr(), x_dtype=0)
        args = _ext.LinearFp8Args(abi_version=_ext.ABI_VERSION, weight=w.data_ptr(), weight_scale=ws.data_ptr(), y=y.data_ptr(), y_dtype=0, m=m,
                                  k=k, n=n, x_stride=k, weight_stride=k, weight_scale_stride=ws.stride(0), y_stride=n, **of_x)
        whole, required = lib.h3a_linear_fp8_workspace_size(ctypes.byref(args)), lib.h3a_linear_fp8_required_workspace(ctypes.byref(args))
        assert whole > required and (required == 0) == x8
        size = required if short else whole
        room = torch.full((size + 4096,), 91, dtype=torch.uint8, device=DEV)
        args.workspace, args.workspace_bytes = room.data_ptr(), size
        assert lib.h3a_linear_fp8(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == _ext.H3A_OK
        _check(y[:m], False, q, s, w, ws, None)
        assert (y[m:] == 7).all() and (room[size:] == 91).all()
        if not short:
            assert torch.equal(y[:m], fused_linear_fp8(q, w, ws, x_scale=s))


def test_more_than_2_31_values():
    # rows far behind 2^31 bytes of every operand, against the same rows alone
    m, k, n = 140_000, 16_000, 15_504
    x = torch.empty((m, k), dtype=BF16, device=DEV)
    x[:] = _activations(1, k, 1)
    x[-300:] = _activations(300, k, 2)
    q, s = quantize_fp8(x)
    _same(q[-300:], s[-300:], x[-300:])
    del x
    w, ws = quantize_fp8_weight(_randn(n, k, seed=3, scale=k**-0.5))
    y = fused_linear_fp8(q, w, ws, x_scale=s)
    last = fused_linear_fp8(q[-256:].clone(), w, ws, x_scale=s[-256:].clone())
    # (other tiles sum in another order: one rounding apart at most)
    assert ((y[-256:].float() - last.float()).abs() <= 2.0**-7 * last.float().abs() + 1e-3).all()
    h, hs = fused_linear_fp8(q[:, :272], w[:, :272], ws[:, :3], x_scale=s[:, :3], quantize=True)
    h2, hs2 = fused_linear_fp8(q[-256:, :272], w[:, :272], ws[:, :3], x_scale=s[-256:, :3], quantize=True)
    # (in 8 bits a sum next to the middle between two values takes another one, a step of
    # 2^-3 away: sums 2^-10 apart do so for 2^-7 of the values, sqrt(2^-7) 2^-3 of the norm)
    a, b = dequantized(h[-256:], hs[-256:]), dequantized(h2, hs2)
    assert (a - b).norm() < 0.02 * b.norm()
    rows = fused_rmsnorm_modulate_fp8(y, torch.ones(n, device=DEV), torch.zeros(1, n, device=DEV), torch.zeros(1, n, device=DEV),
                                      torch.zeros(1, dtype=torch.int64, device=DEV), EPS)
    alone = fused_rmsnorm_modulate_fp8(y[-9:].clone(), torch.ones(n, device=DEV), torch.zeros(1, n, device=DEV), torch.zeros(1, n, device=DEV),
                                       torch.zeros(1, dtype=torch.int64, device=DEV), EPS)
    assert all(torch.equal(a[-9:].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(rows, alone))


def test_a_wide_weight():
    # over 2^31 bytes of weight: rows of it far behind
    n, k = 70_000, 32_000
    w = torch.zeros((n, k), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    few, fs = quantize_fp8_weight(_randn(256, k, seed=1, scale=k**-0.5))
    at = (n // 128 - 2) * 128
    w.view(torch.uint8)[at : at + 256] = few.view(torch.uint8)
    ws = torch.full((-(-n // 128), k // 128), 127, dtype=torch.uint8, device=DEV)
    ws[at // 128 : at // 128 + 2] = fs.view(torch.uint8)
    for m in (5, 40):
        q, s = quantize_fp8(_activations(m, k, 2))
        y = fused_linear_fp8(q, w, ws.view(torch.float8_e8m0fnu), x_scale=s)
        _check(y[:, at : at + 256], False, q, s, few, fs, None)
        assert (y[:, :at] == 0).all()
