"""Training operators at the edges of their domain: masks that outweigh the scores, extreme
values, plans and calls that a program can get wrong."""

from __future__ import annotations

import pytest
import torch

import crumpet_b200 as crumpet
from test_training_gpu import BF16, F16, F32, TOL, attention64, attention_case, rel

pytestmark = pytest.mark.gpu


def attention_both(c, grad=None, **place):
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    place = dict(c["place"], **place)
    return (crumpet.swin_window_attention_train(c["qkv"], c["table"], buckets, **place),
            *crumpet.swin_window_attention_backward(c["grad"] if grad is None else grad, c["qkv"],
                                                    c["table"], buckets, **place))


def attention_wide(c):
    qkv = c["qkv"].double().requires_grad_(True)
    table = c["table"].double().requires_grad_(True)
    out = attention64(qkv, table, c["index"], c["mask"], c["scale"])
    return (out.detach(), *torch.autograd.grad(out, (qkv, table), c["grad"].double()))


# Scores reach 2^10: the product, its sums with bias and mask, and the row's log-sum-exp each
# round them to 2^-14 or finer in fp32, so p and ds are off by at most 4 * 2^-14 (relative); 1e-3
# on top of the tolerances of check_attention.  fp32: the split products' 2^-22 of 2^10, within it.
@pytest.mark.parametrize("shift", [(2, 0, 0), (2, 2, 0), (0, 2, 2), (2, 2, 2)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_mask_is_added_once(dtype, shift):
    """Scores several hundred apart: two tokens on different sides of one, two or three seams
    have one -100 between them (16 channels: -100 / scale is exact in every type)."""
    c = attention_case((4, 4, 4), (2, 2, 2), shift, 2, 2, 16, dtype, F32)
    c["qkv"][:, :, :2] *= 10
    got, want = attention_both(c), attention_wide(c)
    for a, b, tol in zip(got, want, (1.5 * TOL[dtype], TOL[dtype], TOL[F32])):
        assert torch.isfinite(a.float()).all()
        assert rel(a, b) <= tol + 1e-3


@pytest.mark.parametrize("scale", [2.0 ** -8, 1e-3, 1e-5])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_attention_small_scales(dtype, scale):
    """A scale too small for the mask and the padding to be divided by it in the element type
    (27 tokens: padded keys).  Queries and keys are larger by as much: scores of a usual size."""
    c = attention_case((3, 3, 3), (2, 2, 2), (1, 1, 1), 1, 2, 16, dtype, F32)
    c["qkv"][:, :, :2] *= (0.25 / scale) ** 0.5
    c["scale"] = scale
    got, want = attention_both(c, scale=scale), attention_wide(c)
    for a, b, tol in zip(got, want, (1.5 * TOL[dtype], TOL[dtype], TOL[F32])):
        assert torch.isfinite(a.float()).all()
        assert rel(a, b) <= tol


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_attention_mask_is_100_at_32_channels(dtype):
    """-100 / scale is not a number of the element type at scale 32^-1/2.  The mask's weight shows
    where the scores make up for it: all queries are one vector, and keys on one side of the
    seam score 100 (to rounding) above the others, so both sides weigh about the same for
    queries of the other side.  A mask off by e changes the odds by exp(e); one 16-bit number
    is off by 0.3 in bf16 and 0.03 in fp16, the product of two by at most 2^-7 and 2^-11."""
    c = attention_case((2, 4, 4), (1, 2, 1), (0, 2, 0), 1, 1, 32, dtype, F32)
    h = (torch.arange(32, device="cuda") // 4 % 4) >= 2  # the rolled side of the last window
    c["qkv"][:, :, 0] = 4.0
    c["qkv"][:, :, 1] = 0.0
    c["qkv"][:, h, 1] = 4.4219  # 32 * 4 * 4.42 / sqrt 32 = 100.06
    c["table"].zero_()
    got, want = attention_both(c)[0], attention_wide(c)[0]
    off = {BF16: 2.0 ** -7, F16: 2.0 ** -11}[dtype]
    assert rel(got, want) <= TOL[dtype] + off


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_gradient_off_16_bytes(dtype):
    """A gradient off 16-byte boundaries gives what an aligned one does: the kernels are those of
    the forward's qkv."""
    c = attention_case((3, 4, 5), (2, 1, 1), (1, 0, 0), 1, 2, 16, dtype, F32)
    off = torch.empty(c["grad"].numel() + 1, dtype=dtype, device="cuda")[1:].view(c["grad"].shape)
    off.copy_(c["grad"])
    assert off.data_ptr() % 16
    assert all(torch.equal(a, b) for a, b in zip(attention_both(c, grad=off), attention_both(c)))
