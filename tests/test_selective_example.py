"""The example model of selective scan blocks: training lowers its loss, and tokens one by one give what a whole row gives."""
import importlib.util
import sys
from pathlib import Path

import pytest
import torch

_PATH = Path(__file__).resolve().parent.parent / "bayes-ssm_amd" / "examples" / "selective_lm.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("selective_lm", _PATH)
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


def _learns(example, device, dtype):
    torch.manual_seed(1)
    vocabulary = 53
    model = example.SelectiveLM(vocabulary, width=64, blocks=2, heads=2, values=16, n=16).to(device, dtype)
    optimizer = torch.optim.AdamW(model.parameters(), lr=5e-3)
    losses = []
    for _ in range(30):
        tokens = torch.randint(0, vocabulary, (4, 33)).to(device)
        losses.append(example.train_step(model, optimizer, tokens, *example.teach(tokens, vocabulary)).item())
    assert sum(losses[-5:]) < 0.7 * sum(losses[:5])
    return model, vocabulary


def _steps_follow(example, model, vocabulary, device, tolerance):
    prompts = torch.randint(0, vocabulary, (3, 21)).to(device)
    lengths = torch.tensor([21, 9, 1], device=device)
    more = torch.randint(0, vocabulary, (3, 5)).to(device)
    with torch.no_grad():
        _, states = model(prompts, lengths)
        for k in range(5):
            got, states = model.step(more[:, k], states)
            for row, n in enumerate(lengths.tolist()):
                whole, _ = model(torch.cat((prompts[row, :n], more[row, :k + 1]))[None])
                scale = whole[0, -1].float().abs().max()
                assert (got[row].float() - whole[0, -1].float()).abs().max() <= tolerance * scale
    answer = example.generate(model, prompts, lengths, 4)
    assert answer.shape == (3, 4) and 0 <= answer.min() and answer.max() < vocabulary


def test_example_cpu(example):
    model, vocabulary = _learns(example, "cpu", torch.float32)
    _steps_follow(example, model, vocabulary, "cpu", 1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_gpu(example, dtype):
    model, vocabulary = _learns(example, "cuda", dtype)
    # bfloat16: a dozen roundings of 2^-9 on either way, which do not add up in phase; float32: sums of a few hundred terms.
    _steps_follow(example, model, vocabulary, "cuda", 1e-4 if dtype == torch.float32 else 6e-2)
