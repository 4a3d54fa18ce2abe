"""token_logprobs of the heads' linear layers beside their forward."""
import pytest
import torch

from quamba_amd import W4A8B16O16Linear, W8A8B16O16Linear, ops

pytestmark = pytest.mark.gpu


def _layers(dev, out):
    torch.manual_seed(out)
    layer = torch.nn.Linear(256, out, bias=False).half().to(dev)
    return [W8A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217)), W4A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217))]


@pytest.mark.parametrize("out", [500, 1003, 1024])
@pytest.mark.parametrize("lead", [(1,), (1, 1), (2,), (2, 9)])
def test_more_alternatives_are_those_of_forward(dev, out, lead):
    """bit for bit, for one row too, which forward takes through a product of its own"""
    for head in _layers(dev, out):
        for seed in range(4):
            g = torch.Generator().manual_seed(seed)
            x = torch.randint(-127, 128, (*lead, 256), generator=g, dtype=torch.int8).to(dev)
            tokens = torch.randint(0, out, lead, generator=g).to(dev)
            got, want = head.token_logprobs(x, tokens, top=7), ops.token_logprobs(head(x), tokens, top=7)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (type(head).__name__, seed)


def test_no_rows(dev):
    for head in _layers(dev, 500):
        x, tokens = torch.zeros(2, 0, 256, dtype=torch.int8, device=dev), torch.zeros(2, 0, dtype=torch.int64, device=dev)
        for top in (1, 5):
            got = head.token_logprobs(x, tokens, top)
            assert got.logprobs.shape == (2, 0) and got.top_tokens.shape == (2, 0, top)
