"""Beam selection of the int8 heads with a scale for each row: the logits are those of the product with these scales."""
import pytest
import torch

from quamba_amd import W4A8B16O16Linear, W8A8B16O16Linear, ops

pytestmark = pytest.mark.gpu


def heads(dev, out):
    torch.manual_seed(out)
    layer = torch.nn.Linear(256, out, bias=False).half().to(dev)
    return [cls.from_fp16(layer, torch.tensor(0.0217)) for cls in (W8A8B16O16Linear, W4A8B16O16Linear)]


def logits_of(head, x2d, scales):
    if isinstance(head, W4A8B16O16Linear):
        y = ops.w4a8o16_gemm(x2d, head.weight, scales, head.s_channel, head.s_group, head.workspace, x2d.shape[0], head.size_n, head.size_k)
    else:
        y = torch.empty((x2d.shape[0], head.weight.shape[1]), dtype=torch.float16, device=x2d.device)
        ops.scaled_mm_dq(y, x2d, head.weight, scales, head.b)
    return y[:, :head.out_features]


@pytest.mark.parametrize("out", [500, 1003])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 5), (2, 3), (7, 4)])
def test_a_scale_for_each_row(dev, out, batch, beams):
    for head in heads(dev, out):
        x = torch.randint(-127, 128, (batch, beams, 256), dtype=torch.int8, device=dev)
        scores, x_scale = torch.randn(batch, beams, device=dev), 0.01 + 0.03 * torch.rand(batch, beams, device=dev)
        done = torch.rand(batch, beams, device=dev) < 0.3
        logits = logits_of(head, x.view(-1, 256), x_scale.view(-1)).reshape(batch, beams, out)
        # (a row's scale alone sets its logits apart: those of the layer's own scale, times the quotient, to within their roundings of half a step each)
        own = logits_of(head, x.view(-1, 256), torch.full((batch * beams,), 0.0217, device=dev)).reshape(batch, beams, out).double()
        assert ((logits.double() - own * (x_scale.double() / 0.0217)[..., None]).abs() <= logits.double().abs() * (2.0 ** -10 + 2.0 ** -20) + 2.0 ** -22).all()
        for mask in (None, done):
            got, want = head.beam_search_step(x, scores, 5, mask, x_scale=x_scale), ops.beam_search_step(logits, scores, 5, mask)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            # scales, scores and states as they lie
            got = head.beam_search_step(x, scores.t().contiguous().t(), 5, mask, x_scale=x_scale.t().contiguous().t())
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scales_that_are_refused(dev):
    for head in heads(dev, 500):
        x, scores = torch.zeros(2, 3, 256, dtype=torch.int8, device=dev), torch.zeros(2, 3, device=dev)
        for shape in ((6,), (3, 2), (2,), (2, 3, 1), (1, 3), ()):
            with pytest.raises(RuntimeError, match="x_scale must have shape"):
                head.beam_search_step(x, scores, 4, x_scale=torch.ones(shape, device=dev))
