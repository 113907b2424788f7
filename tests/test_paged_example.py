"""The paged operators together: the example decoder (examples/paged_beams.py)
against the CPU oracle at the same context length, by the parity rule of the
2-layer models (tests/test_gpu_engine.py)."""

import importlib.util

import numpy as np
import pytest

from conftest import PKG
from oracle.cpu_decoder import OracleDecoder
from runtime import synthetic
from test_gpu_engine import assert_logits_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_beams", PKG / "examples" / "paged_beams.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("name", ["tiny-qwen", "tiny-llama"])
def test_chunks_and_decode_match_the_oracle(example, name):
    import torch

    model = synthetic.build(name, seed=31)
    ids = synthetic.prompt_ids(model.shape.vocab, 150, seed=4)
    decoder = example.PagedDecoder(model, 3, 256, 12)
    oracle = OracleDecoder(model, context_length=256)
    ref = [oracle.step(t, p) for p, t in enumerate(ids)]
    dev = lambda x: torch.tensor(x, device="cuda")  # noqa: E731
    got = decoder.prefill(1, dev(ids[:130]), chunk=70)
    assert_logits_close(got.cpu().numpy(), ref[129], "chunked prompt")
    # its fork decodes on while the first, shorter one takes another chunk
    decoder.cache.fork(decoder.ints([1]), decoder.ints([2]), decoder.ints([100]))
    rows = decoder.step([2, 1], [30, 1], dev(list(ids[100:130]) + [ids[130]]))
    assert_logits_close(rows[0].cpu().numpy(), ref[129], "fork's chunk")
    assert_logits_close(rows[1].cpu().numpy(), ref[130], "decode")
    decoder.cache.free(decoder.ints([2]))
    decoder.cache.compact()
    for p in range(131, 150):
        got = decoder.step([1], [1], dev([ids[p]]))
    assert_logits_close(got[0].cpu().numpy(), ref[149], "after the compaction")
    decoder.cache.status()


def test_beams_share_their_prompt(example):
    """Each beam's tokens are those it would decode alone, and the beams hold
    the prompt's whole pages once."""
    import torch

    model = synthetic.build("tiny-qwen", seed=31)
    prompt = torch.tensor(synthetic.prompt_ids(model.shape.vocab, 200, seed=5), device="cuda")
    decoder = example.PagedDecoder(model, 5, 256, 40)
    tokens, scores = example.beams(decoder, prompt, 4, 6, swap_at=100)
    decoder.cache.status()
    table = decoder.cache.table.cpu().numpy()
    assert len({tuple(r[:3]) for r in table[1:5]}) == 1 and len(set(table[1:5, 3])) == 4
    for beam in range(4):
        alone = example.PagedDecoder(model, 1, 256, 8)
        logits = alone.prefill(0, prompt)
        total = float(torch.log_softmax(logits.double(), 0)[tokens[beam, 0]])
        for t in range(1, 6):
            step = alone.step([0], [1], tokens[beam, t - 1: t])
            lp = torch.log_softmax(step[0].double(), 0)
            total += float(lp[tokens[beam, t]])
            assert float(lp.max() - lp[tokens[beam, t]]) < 2e-2  # the best, or as good to rounding
        assert abs(total - float(scores[beam])) < 5e-2


def test_beams_permuted(example):
    """Forks whose sources are destinations, in a search that swaps beams."""
    import torch

    model = synthetic.build("tiny-llama", seed=3)
    prompt = torch.tensor(synthetic.prompt_ids(model.shape.vocab, 70, seed=6), device="cuda")
    decoder = example.PagedDecoder(model, 6, 128, 40)
    tokens, scores = example.beams(decoder, prompt, 5, 12, swap_at=3)
    decoder.cache.status()
    assert tokens.shape == (5, 12) and bool(torch.isfinite(scores).all())
    refs = decoder.cache.refs.cpu().numpy()
    table = decoder.cache.table.cpu().numpy()
    assert np.array_equal(refs, np.bincount(table[table >= 0], minlength=len(refs)))


def test_command_runs(example, capsys):
    example.main(["--prompt", "100", "--beams", "3", "--new", "10"])
    assert "3 beams" in capsys.readouterr().out
