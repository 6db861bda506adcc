"""project_joiner_fp8 where all logits of a row are far below zero: biases of the type's lowest value
in place of a mask, in every kernel and split of the vocabulary."""
import math

import pytest
import torch

import optimized_transducer_amd as ot

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("rows,D,V", [(3, 256, 40), (20, 512, 500), (2000, 112, 500), (1500, 256, 501), (40000, 384, 500),
                                      (1700, 512, 1021), (2111, 640, 1001), (9000, 1040, 1025), (5000, 2064, 130), (70000, 128, 100)])
@pytest.mark.parametrize("fill", [LOWEST, -3e38, -1e32, -2e30, -9e29, 1e30, 3e38, 3.3e38, -LOWEST])
def test_denominators_of_rows_far_from_zero(rows, D, V, fill, device):
    """A bias so large that the products vanish beside it: the denominator of V equal logits is
    bias + log V, which float32 rounds to the bias; two values apart by more than that leave the larger."""
    g = torch.Generator(device=device).manual_seed(rows)
    x, xs = ot.quantize_blocks(torch.randn((rows, D), device=device, generator=g))
    w, ws = ot.quantize_blocks(torch.randn((V, D), device=device, generator=g) / math.sqrt(D), 128)
    bias = torch.full((V,), fill, device=device)
    for dtype in (torch.float32, torch.bfloat16):
        logits, den = ot.project_joiner_fp8(x, xs, w, ws, bias, logits_dtype=dtype)
        assert torch.equal(logits, bias.to(dtype).expand(rows, V))
        assert torch.equal(den, bias[:1].expand(rows))
    bias[V // 2] = fill * 0.5 if fill < 0 else fill
    bias[V - 1] = -math.inf
    _, den = ot.project_joiner_fp8(x, xs, w, ws, bias)
    assert torch.equal(den, bias[V // 2:V // 2 + 1].expand(rows))
    bias.fill_(LOWEST)
    bias[V - 1] = 0.0  # one entry that is not masked
    logits, den = ot.project_joiner_fp8(x, xs, w, ws, bias)
    assert (den - logits[:, V - 1]).abs().max() <= 2.0 ** -21 * (1 + float(logits[:, V - 1].abs().max()))
