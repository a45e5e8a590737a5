"""The serving operators in a run together, as a decode loop makes it.

* Two layers of a bounded cache over many steps: write, attend (gathering
  weights), evict, each step's operators compared with their definitions in 64
  bits on the state that the step before left; the same steps replayed from one
  captured graph give the same bits.
* The decoder step's logits through process_logits: without penalties the
  tokens are the resident epoch's; with a repetition penalty and a mask, those of
  the formula.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from cruise_amd.runtime import pack_feed, tiling_bytes
from kv_ops_reference import attention, evict, process_logits, rotated, weights_after, wide, write_tolerance
from oracle.controller import control_input_elements
from oracle.weights import generate_weights
from oracle.workloads import C1, identity_table, slot_of
from parity import make_runtime

pytestmark = pytest.mark.gpu
LAYERS, ROWS, HEADS, KV_HEADS, D, BLOCK, WIDTH, BUDGET, RECENT, SINKS = 2, 3, 14, 2, 128, 16, 5, 48, 12, 2


class Loop:
    """Caches in the decoder-step layout [layers, pages, block, kv_heads, head_dim]
    and the device state of a decode loop over them."""

    def __init__(self, dtype):
        gen = torch.Generator().manual_seed(31)
        pages = ROWS * WIDTH + 1
        self.keys = torch.zeros(LAYERS, pages, BLOCK, KV_HEADS, D, dtype=dtype, device="cuda")
        self.values = torch.zeros_like(self.keys)
        self.weights = torch.zeros(LAYERS, pages, KV_HEADS, BLOCK, device="cuda")
        self.positions = torch.full((LAYERS, pages, KV_HEADS, BLOCK), -1, dtype=torch.int32, device="cuda")
        self.table = torch.randperm(pages, generator=gen)[: ROWS * WIDTH].int().view(ROWS, WIDTH).cuda()
        self.lengths = torch.tensor([0, 20, 45], dtype=torch.int32, device="cuda")
        self.next = self.lengths.long()
        for r, n in enumerate(self.lengths.tolist()):  # rows that have begun: random tokens in order
            for j in range(n):
                page, at = int(self.table[r, j // BLOCK]), j % BLOCK
                self.keys[:, page, at] = torch.randn(LAYERS, KV_HEADS, D, generator=gen).to(dtype).cuda()
                self.values[:, page, at] = torch.randn(LAYERS, KV_HEADS, D, generator=gen).to(dtype).cuda()
                self.positions[:, page, :, at] = j
        self.inv_freq = (1e4 ** (-torch.arange(0, D, 2).double() / D)).float().cuda()
        self.norms = [(1 + 0.1 * torch.randn(D, generator=gen)).to(dtype).cuda() for _ in range(2)]
        self.qkv = torch.zeros(LAYERS, ROWS, HEADS + 2 * KV_HEADS, D, dtype=dtype, device="cuda")
        self.out = torch.zeros(LAYERS, ROWS, HEADS, D, dtype=dtype, device="cuda")

    def new_tokens(self, step):
        gen = torch.Generator().manual_seed(1000 + step)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=gen))

    def write_args(self, layer, slots):
        q, k, v = self.qkv[layer].split([HEADS, KV_HEADS, KV_HEADS], dim=1)
        return dict(q=q, k=k, v=v, positions=self.next, slots=slots, key_cache=self.keys[layer], value_cache=self.values[layer],
                    inv_freq=self.inv_freq, q_norm=self.norms[0], k_norm=self.norms[1])

    def slots(self):
        pages = self.table.gather(1, (self.lengths // BLOCK).long()[:, None])[:, 0]
        return pages * BLOCK + self.lengths % BLOCK

    def step(self, check=None):
        slots = self.slots()
        self.lengths += 1
        new = None
        for layer in range(LAYERS):
            if check:
                check.before(self, layer)
            q = ops.kv_write(**self.write_args(layer, slots), weight_cache=self.weights[layer], position_cache=self.positions[layer])
            if check:
                check.written(self, layer, slots, q)
            ops.kv_attention(q, self.keys[layer], self.values[layer], self.table, self.lengths, weight_cache=self.weights[layer],
                             out=self.out[layer])
            if check:
                check.attended(self, layer, q)
            if check:
                check.evicting(self, layer)
            new = ops.kv_evict(self.keys[layer], self.values[layer], self.table, self.lengths, self.next + 1, self.weights[layer],
                               self.positions[layer], budget=BUDGET, recent=RECENT, sinks=SINKS)
            if check:
                check.evicted(self, layer, new)
        self.lengths.copy_(new)
        self.next += 1

    def state(self):
        return (self.keys, self.values, self.weights, self.positions, self.lengths, self.next, self.out)


class Check:
    def before(self, s, layer):
        self.was = [t[layer].clone() for t in (s.keys, s.values, s.weights, s.positions)]

    def written(self, s, layer, slots, q):
        a = s.write_args(layer, slots)
        for x, norm, got in ((a["q"], a["q_norm"], q), (a["k"], a["k_norm"], s.keys[layer].flatten(0, 1)[slots.long()])):
            ref, size = rotated(x, norm, 1e-6, s.next, s.inv_freq)
            assert (np.abs(wide(got) - ref) <= write_tolerance(ref, size, x.dtype, D)).all()
        assert torch.equal(s.values[layer].flatten(0, 1)[slots.long()], a["v"])
        for now, was in ((s.keys, self.was[0]), (s.values, self.was[1])):
            now = now[layer].flatten(0, 1).clone()
            now[slots.long()] = was.flatten(0, 1)[slots.long()]
            assert torch.equal(now, was.flatten(0, 1))
        self.was = [t[layer].clone() for t in (s.keys, s.values, s.weights, s.positions)]

    def attended(self, s, layer, q):
        ref, tol, p = attention(q, s.keys[layer], s.values[layer], s.table, s.lengths)
        assert (np.abs(wide(s.out[layer]) - ref) <= tol).all()
        ref, tol = weights_after(self.was[2], p, KV_HEADS)
        assert (np.abs(wide(s.weights[layer]) - ref) <= tol).all()
        # every query head of a row hands out a weight of one
        given = (s.weights[layer] - self.was[2]).double().sum()
        assert abs(float(given) - ROWS * HEADS) < 1e-3

    def evicting(self, s, layer):
        self.ref = evict(s.keys[layer], s.values[layer], s.weights[layer], s.positions[layer], s.table, s.lengths, s.next + 1, BUDGET, RECENT, SINKS)

    def evicted(self, s, layer, new):
        for x, y in zip((s.keys[layer], s.values[layer], s.weights[layer], s.positions[layer], new), self.ref):
            assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bounded_cache_over_many_steps(dtype):
    loop, check = Loop(dtype), Check()
    for step in range(40):
        loop.new_tokens(step)
        loop.step(check)
    assert loop.lengths.tolist() == [40, BUDGET, BUDGET] and loop.next.tolist() == [40, 60, 85]
    # the newest tokens and the first ones are there, for every layer and KV head
    for r, n in ((1, 60), (2, 85)):
        held = loop.positions[:, loop.table[r].long()].transpose(2, 1).flatten(2)
        for layer in range(LAYERS):
            for g in range(KV_HEADS):
                have = set(held[layer, g].tolist())
                assert {0, 1} | set(range(n - RECENT + 1, n)) <= have


def test_captured_steps_equal_eager_ones():
    eager, captured = Loop(torch.bfloat16), Loop(torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for step in range(12):
        for loop in (eager, captured):
            loop.new_tokens(step)
        eager.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(eager.state(), captured.state()):
            assert torch.equal(x, y)


def test_two_loops_on_two_streams():
    """Two decode loops at the same time, each on a stream of its own, and their
    logits beside them: the same bits as one after the other."""
    alone, together = ([Loop(torch.bfloat16), Loop(torch.float32)] for _ in range(2))
    gen = torch.Generator().manual_seed(32)
    logits = [torch.randn(5, 30011, generator=gen).cuda() for _ in range(2)]
    options = dict(history=torch.randint(0, 30011, (5, 4000), generator=gen).cuda(),
                   history_lengths=torch.full((5,), 4000, dtype=torch.int32, device="cuda"), repetition=torch.full((5,), 1.3, device="cuda"))
    want = [ops.process_logits(x, **options) for x in logits]
    for step in range(10):
        for loop in alone:
            loop.new_tokens(step)
            loop.step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for step in range(10):
        for loop, stream, x in zip(together, streams, logits):
            with torch.cuda.stream(stream):
                loop.new_tokens(step)
                loop.step()
                got.append(ops.process_logits(x, **options))
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a.state(), b.state()))
    for i, (out, tokens) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(tokens, want[i % 2][1])


def test_operator_timing_command():
    """The command that times the operators runs them all at an odd size."""
    from cruise_amd.opbench import serving

    times = serving(3, 301, 2)
    assert [name for name, _, _ in times] == ["kv_write", "kv_attention", "kv_attention + weights", "kv_evict", "process_logits"]
    assert all(us > 0 and nbytes > 0 for _, us, nbytes in times)


def decode(rt, steps, choose):
    """Greedy decoding by decoder steps on caches of the caller's, one token of every row a step."""
    g, d = C1.geometry, C1.dims
    B = g.batch
    table = identity_table(B, g.blocks_per_row)
    shape = (d.num_layers, g.physical_blocks, g.block_size, d.num_kv_heads, d.head_dim)
    keys, values = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    logits = torch.zeros(B, d.vocab, device="cuda")
    position, tokens = np.zeros(B, dtype=np.int64), np.arange(5, 5 + B, dtype=np.int64)
    history = torch.zeros(B, steps + 1, dtype=torch.int64, device="cuda")
    history[:, 0] = torch.from_numpy(tokens)
    for n in range(1, steps + 1):
        slots = np.array([slot_of(table, r, int(position[r]), g.block_size) for r in range(B)], dtype=np.int32)
        rt.decoder_step(history[:, n - 1], position, (position + 1).astype(np.int32), keys, slots, np.ones(B, np.int32), table, values,
                        logits, torch.zeros(B, dtype=torch.int64, device="cuda"))
        history[:, n] = choose(logits, history, n)
        position += 1
    return history


def test_decoder_step_logits():
    weights = generate_weights(C1.dims, C1.seed)
    rt = make_runtime(C1, weights)
    try:
        g, steps = C1.geometry, 8
        B = g.batch
        plain = decode(rt, steps, lambda logits, history, n: ops.process_logits(logits)[1])
        table = identity_table(B, g.blocks_per_row)
        tokens, positions = np.arange(5, 5 + B, dtype=np.int64), np.zeros(B, dtype=np.int64)
        slots = np.array([slot_of(table, r, 0, g.block_size) for r in range(B)], dtype=np.int32)
        control = np.zeros(control_input_elements(B), dtype=np.int32)
        control[0] = steps
        control[1 : 1 + B] = C1.eos
        control[3 + B :] = np.arange(1, B + 1)
        chosen, _ = rt.proc(pack_feed(tokens, positions, np.ones(B, np.int32), slots, np.ones(B, np.int32), table, tiling_bytes(), control))
        assert C1.eos not in chosen
        np.testing.assert_array_equal(plain[:, 1:].cpu().numpy().T, chosen)

        allowed = torch.randint(-(2**31), 2**31, (B, C1.dims.vocab // 32), generator=torch.Generator().manual_seed(3)).int().cuda()
        rep = torch.full((B,), 1.7, device="cuda")

        def constrained(logits, history, n):
            options = dict(history=history, history_lengths=torch.full((B,), n, dtype=torch.int32, device="cuda"), repetition=rep,
                           allowed=allowed)
            before = logits.clone()
            out, picked = ops.process_logits(logits, **options, out=logits)
            ref, want = process_logits(before, np.float32, **options)
            np.testing.assert_array_equal(wide(out), ref.astype(np.float64))
            np.testing.assert_array_equal(picked.cpu().numpy(), want)
            return picked

        history = decode(rt, steps, constrained)
        for r in range(B):
            for token in history[r, 1:].tolist():
                assert int(allowed[r, token // 32]) >> (token % 32) & 1
    finally:
        rt.close()
