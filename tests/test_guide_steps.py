"""The decode step that the guides at the repository's root show, run on the host
with stand-ins for the operators: every layer writes, attends and evicts under the
same lengths, and only the step after sees the evicted ones."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from cruise_amd import ops

ROOT = Path(__file__).resolve().parents[1]
STEPS = [block for guide in sorted(ROOT.glob("*.md")) for block in re.findall(r"```python\n(.*?)```", guide.read_text(), re.S)
         if "ops.kv_evict(" in block]
LAYERS, BLOCK, BUDGET = 3, 4, 1024


def test_a_guide_shows_the_step():
    assert STEPS


@pytest.mark.parametrize("step", STEPS)
def test_layers_share_their_lengths(step, monkeypatch):
    seen = []

    def note(name, lengths):
        seen.append((name, lengths.tolist()))

    def kv_write(q, k, v, positions, slots, keys, values, inv_freq, **more):
        note("write", slots)
        assert more["weight_cache"].shape == more["position_cache"].shape == (4, 1, BLOCK) and keys.shape == (4, BLOCK, 1, 64)
        return q

    def kv_attention(q, keys, values, table, lengths, **more):
        note("attend", lengths)
        return q

    def kv_evict(keys, values, table, lengths, next_positions, weights, held, *, budget, recent, sinks, max_length):
        note("evict", lengths)
        assert budget == BUDGET and next_positions.tolist() == [2001, 8]
        return lengths.clamp(max=budget)

    for f in (kv_write, kv_attention, kv_evict):
        monkeypatch.setattr(ops, f.__name__, f)
    monkeypatch.setattr(ops, "process_logits", lambda logits, **more: (logits, logits.argmax(1)))
    table = torch.arange(2 * 300, dtype=torch.int32).view(2, 300)
    names = dict(
        key_cache=torch.zeros(LAYERS, 4, BLOCK, 1, 64), value_cache=torch.zeros(LAYERS, 4, BLOCK, 1, 64),
        weights=torch.zeros(LAYERS, 4, 1, BLOCK), held=torch.zeros(LAYERS, 4, 1, BLOCK, dtype=torch.int32), block_table=table,
        lengths=torch.tensor([BUDGET, 7], dtype=torch.int32), positions=torch.tensor([2000, 7]), longest=1200, block=BLOCK, layers=LAYERS,
        hidden=torch.zeros(2, 8), inv_freq=torch.zeros(32), q_norms=[None] * LAYERS, k_norms=[None] * LAYERS,
        project=lambda layer, hidden: (torch.zeros(2, 1, 64),) * 3, finish=lambda layer, hidden, out: hidden, head=lambda hidden: hidden,
        tokens_so_far=None, counts=None, prompts=None, rep=None, grammar=None)
    exec(step, names)
    slots, grown = [BUDGET // BLOCK * BLOCK, 300 * BLOCK + 7], [BUDGET + 1, 8]  # row 1's table begins at page 300
    assert seen == [("write", slots), ("attend", grown), ("evict", grown)] * LAYERS
    assert names["lengths"].tolist() == [BUDGET, 8] and names["positions"].tolist() == [2001, 8]
    assert names["tokens"].shape == (2,)
