"""The example decoder stack: attention on the paged cache and the split FFN together, through
prefill, fork, decode, drop, compact and decode again."""
from __future__ import annotations

import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("decoder_layers", ROOT / "examples" / "decoder_layers.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("prompt,samples", [(70, 3), (16, 2)])
def test_samples_of_a_prompt_agree_and_survive_compaction(cuda, prompt, samples):
    import torch
    example = load()
    r = example.run(layers=2, prompt=prompt, samples=samples, steps=6, d_ff=128)
    x = r["samples"].view(2, samples, -1)
    assert torch.isfinite(x).all() and (x[0, 0] != x[1, 0]).any()
    for other in range(1, samples):  # the same tokens after the same shared pages: the same bits
        assert torch.equal(x[:, 0], x[:, other])
    assert torch.isfinite(r["last"]).all() and r["lengths"].tolist() == [prompt + 12, max(1, prompt // 3) + 12]
    held = [p for row, n in zip(r["tables"].tolist(), r["lengths"].tolist()) for p in row[:-(-n // 16)]]
    assert len(set(held)) == len(held)
    # one sample from the start, never forked nor compacted, ends in the same place (1 in 100: torch's
    # products may sum in another order for another batch)
    alone = example.run(layers=2, prompt=prompt, samples=1, steps=6, d_ff=128)
    assert (alone["last"].double() - r["last"].double()).norm() <= 1e-2 * r["last"].double().norm()
