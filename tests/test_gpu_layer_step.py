"""A layer's decode step as a caller's loop runs it: norms to 8 bits, the projection
of q, k and v, the cache write, attention behind a shared prefix, eviction of the own
slots, the output projection; step by step against 64 bits, and captured."""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import wide
from layer_ops_reference import STEP, norms, prefix_attention, product

pytestmark = pytest.mark.gpu
HEADS, KV, D, BLOCK, HIDDEN, ROWS, WIDTH = 8, 2, 64, 16, 512, 5, 3
BUDGET, RECENT = 24, 8


class Loop:
    """One layer, its rows behind a prefix of `prefix` slots that is in the cache already."""

    def __init__(self, prefix, seed, dtype=torch.bfloat16):
        gen = torch.Generator().manual_seed(seed)
        randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        shared = -(-prefix // BLOCK)
        pages = shared + ROWS * WIDTH + 1
        self.keys, self.values = randn(pages, BLOCK, KV, D).to(dtype).cuda(), randn(pages, BLOCK, KV, D).to(dtype).cuda()
        self.weights = torch.rand(pages, KV, BLOCK, generator=gen).cuda()
        self.held = torch.full((pages, KV, BLOCK), -1, dtype=torch.int32).cuda()
        order = torch.randperm(pages, generator=gen).int()
        self.prefix_table, self.table = order[:shared].clone().cuda(), order[shared : shared + ROWS * WIDTH].view(ROWS, WIDTH).clone().cuda()
        self.prefix_length = torch.tensor([prefix], dtype=torch.int32).cuda()
        self.lengths = torch.tensor([0, 3, 20, 23, 24], dtype=torch.int32).cuda()
        self.positions = prefix + self.lengths.long()
        vector = lambda n: (1 + 0.1 * randn(n)).to(dtype).cuda()  # noqa: E731
        self.post, self.pre, self.gate, self.bias = vector(HIDDEN), vector(HIDDEN), vector(HIDDEN), vector((HEADS + 2 * KV) * D)
        self.qkv = ops.quantize_rows((randn((HEADS + 2 * KV) * D, HIDDEN) * HIDDEN**-0.5).to(dtype).cuda())
        self.out = ops.quantize_rows((randn(HIDDEN, HEADS * D) * HIDDEN**-0.5).to(dtype).cuda())
        self.inv_freq = (1e4 ** (-torch.arange(0, D, 2).double() / D)).float().cuda()
        self.block, self.residual = randn(ROWS, HIDDEN).to(dtype).cuda(), randn(ROWS, HIDDEN).to(dtype).cuda()

    def state(self):
        return dict(keys=self.keys, values=self.values, weights=self.weights, held=self.held, lengths=self.lengths, positions=self.positions,
                    block=self.block, residual=self.residual)

    def step(self, check=False):
        before = self.residual.clone()
        residual, x, scales = ops.block_norms(self.block, self.residual, post_norm=self.post, gate=self.gate, scale=0.5, pre_norm=self.pre,
                                              quantize=True, residual_out=self.residual)
        qkv = ops.int8_linear(x, *self.qkv, x_scale=scales, bias=self.bias, dtype=self.block.dtype)
        q, k, v = qkv.view(ROWS, HEADS + 2 * KV, D).split([HEADS, KV, KV], dim=1)
        at = self.lengths[:, None] // BLOCK
        slots = self.table.gather(1, at.long())[:, 0] * BLOCK + self.lengths % BLOCK
        q = ops.kv_write(q, k, v, self.positions, slots, self.keys, self.values, self.inv_freq, weight_cache=self.weights,
                         position_cache=self.held)
        grown = self.lengths + 1
        gathered = self.weights.clone() if check else None
        args = (q, self.keys, self.values, self.prefix_table, self.prefix_length, self.table, grown)
        attended = ops.kv_prefix_attention(*args, weight_cache=self.weights, max_length=WIDTH * BLOCK)
        out = ops.int8_linear(attended.flatten(1), *self.out)
        if check:
            self.compare(before, residual, x, scales, qkv, args, attended, gathered, out)
        kept = ops.kv_evict(self.keys, self.values, self.table, grown, self.positions + 1, self.weights, self.held, budget=BUDGET, recent=RECENT,
                            max_length=WIDTH * BLOCK)
        self.block.copy_(out)
        self.lengths.copy_(kept)
        self.positions.add_(1)

    def compare(self, before, residual, x, scales, qkv, args, attended, gathered, out):
        ref, tol, normed, loose = norms(self.block, before, self.pre, self.post, self.gate, scale=0.5)
        assert (np.abs(wide(residual) - ref) <= tol).all()
        steps = wide(scales)[:, None]
        assert (np.abs(wide(x) * steps - normed) <= loose + steps * (0.5 + 254 * STEP)).all()
        ref, tol = product(x.cpu().numpy(), scales.cpu().numpy(), *self.qkv, self.bias, qkv.dtype)
        assert (np.abs(wide(qkv) - ref) <= tol).all()
        ref, tol, given, given_tol = prefix_attention(*args)
        assert (np.abs(wide(attended) - ref) <= tol).all()
        assert (np.abs(wide(self.weights) - wide(gathered) - given) <= given_tol + STEP * (wide(gathered) + given)).all()
        x8, s8 = ops.quantize_rows(attended.flatten(1))
        ref, tol = product(x8.cpu().numpy(), s8.cpu().numpy(), *self.out, None, out.dtype)
        assert (np.abs(wide(out) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("prefix", [0, 7, 96, 1000])
def test_steps(prefix, dtype):
    loop = Loop(prefix, prefix + 1, dtype)
    held_before = loop.held[loop.prefix_table.long()].clone()
    weights_before = loop.weights[loop.prefix_table.long()].clone()
    for _ in range(6):
        loop.step(check=True)
    assert loop.lengths.tolist() == [6, 9, 24, 24, 24]
    # nothing of the prefix was written, weighed or evicted
    assert torch.equal(loop.held[loop.prefix_table.long()], held_before)
    assert torch.equal(loop.weights[loop.prefix_table.long()], weights_before)


def test_pages_of_a_whole_prefix():
    """A prefix of whole pages is what kv_attention sees in front of a row's own pages."""
    loop = Loop(96, 3)
    q = torch.randn(ROWS, HEADS, D, device="cuda").bfloat16()
    args = (q, loop.keys, loop.values, loop.prefix_table, loop.prefix_length, loop.table, loop.lengths)
    both = torch.cat([loop.prefix_table.expand(ROWS, -1), loop.table], dim=1)
    whole = ops.kv_attention(q, loop.keys, loop.values, both, loop.lengths + 96)
    _, tol, _, _ = prefix_attention(*args)
    assert (np.abs(wide(ops.kv_prefix_attention(*args)) - wide(whole)) <= 2 * tol).all()


def test_captured_steps():
    """A captured step, replayed with eager work between, leaves what as many eager ones do."""
    loops = [Loop(300, 5) for _ in range(2)]
    before = {k: v.clone() for k, v in loops[0].state().items()}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        loops[0].step()  # warm: the library's first calls of each kernel
    torch.cuda.synchronize()
    for k, v in loops[0].state().items():
        v.copy_(before[k])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loops[0].step()
    for k, v in loops[0].state().items():
        v.copy_(before[k])
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        loops[1].step()
        torch.cuda.synchronize()
        for k, v in loops[1].state().items():
            assert torch.equal(loops[0].state()[k], v), k


ROOT = Path(__file__).resolve().parents[1]
STEPS = [block for guide in sorted(ROOT.glob("*.md")) for block in re.findall(r"```python\n(.*?)```", guide.read_text(), re.S)
         if "ops.kv_prefix_attention(" in block]


def test_a_guide_shows_the_step():
    assert STEPS


@pytest.mark.parametrize("step", STEPS)
def test_the_guides_step(step):
    """The layer that the guides at the repository's root show does what the loop above does."""
    a, b = Loop(40, 11), Loop(40, 11)
    gen = torch.Generator().manual_seed(12)
    qkv, out = torch.randn((HEADS + 2 * KV) * D, HIDDEN, generator=gen).cuda(), torch.randn(HIDDEN, HEADS * D, generator=gen).cuda()
    a.qkv, a.out = ops.quantize_rows(qkv), ops.quantize_rows(out)
    grown = b.lengths + 1
    slots = b.table.gather(1, (b.lengths[:, None] // BLOCK).long())[:, 0] * BLOCK + b.lengths % BLOCK
    names = dict(qkv_weight=qkv, out_weight=out, block_out=b.block, residual=b.residual, after=b.post, before=b.pre, gate=b.gate, qkv_bias=b.bias,
                 rows=ROWS, heads=HEADS, kv_heads=KV, d=D, positions=b.positions, slots=slots, keys=b.keys, values=b.values, inv_freq=b.inv_freq,
                 prefix_table=b.prefix_table, prefix_length=b.prefix_length, block_table=b.table, grown=grown, prefix_slots=40,
                 longest=WIDTH * BLOCK)
    exec(step, names)
    a.step()
    assert torch.equal(names["block_out"], a.block) and torch.equal(names["residual"], a.residual)


def test_operator_timing_command():
    """The command that times the operators runs them all at an odd size."""
    from cruise_amd.opbench import serving_layer

    times = serving_layer(3, 301, 2)
    assert [name.split()[0] for name, _, _ in times] == ["kv_prefix_attention"] + 2 * ["block_norms"] + 4 * ["int8_linear"]
    assert all(us > 0 and nbytes > 0 for _, us, nbytes in times)
