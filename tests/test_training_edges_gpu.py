"""Training operators at the edges of their domain: masks that outweigh the scores, extreme
values, plans and calls that a program can get wrong."""

from __future__ import annotations

import pytest
import torch

import crumpet_b200 as crumpet
from crumpet_b200 import fused_attention, training
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


BAD_BUCKETS = [
    (BF16, 16, (4, 4, 4)),  # tensor cores
    (F16, 32, (5, 5, 3)),
    (F32, 16, (3, 4, 5)),   # split tf32 products
    (F32, 64, (3, 3, 3)),   # fp32 arithmetic, bias held whole
    (BF16, 128, (8, 8, 9)),  # and tile by tile
]


@pytest.mark.parametrize("dtype,d,win", BAD_BUCKETS, ids=str)
def test_attention_buckets_outside_the_table(dtype, d, win):
    """Buckets outside the table add no bias, in both directions, and are reported."""
    c = attention_case(win, (1, 1, 1), (0, 0, 0), 2, 2, d, dtype, F32)
    rows = c["table"].shape[0]
    c["table"][-1] = 0
    good = crumpet.relative_position_buckets(c["index"], rows)
    last = good.pairs == 3
    zero = good.pairs.masked_fill(last, rows - 1)
    bad = good.pairs.masked_fill(last, rows)
    bad[last & (torch.arange(last.shape[0], device="cuda") % 2 == 0)] = -1

    def run(pairs):
        plan = good._replace(pairs=pairs, index=pairs.long())
        return (crumpet.swin_window_attention_train(c["qkv"], c["table"], plan, **c["place"]),
                *crumpet.swin_window_attention_backward(c["grad"], c["qkv"], c["table"], plan,
                                                        **c["place"]))

    crumpet.device_status(clear=True)
    want = run(zero)
    assert crumpet.device_status() == 0
    got = run(bad)
    assert crumpet.device_status(clear=True) == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("heads", [3, 8])
def test_bias_buckets_outside_the_table(heads, dtype):
    index = torch.arange(64 * 33, device="cuda").view(64, 33) % 40
    plan = crumpet.relative_position_buckets(index, 40)
    table = torch.randn(40, heads, device="cuda").to(dtype)
    want = crumpet.relative_position_bias(table, plan)
    pairs = plan.pairs.clone()
    pairs[5, 7], pairs[63, 32], pairs[0, 0] = 40, -3, 2 ** 31 - 1
    crumpet.device_status(clear=True)
    got = crumpet.relative_position_bias(table, plan._replace(pairs=pairs))
    assert crumpet.device_status(clear=True) == 2
    out = pairs != plan.pairs
    assert torch.equal(got, want.masked_fill(out, 0))


def test_bias_gradient_of_a_plan_that_is_not_one():
    """Places, items and joined buckets outside their tensors are reported and left out."""
    index = torch.arange(64 * 33, device="cuda").view(64, 33) % 40
    plan = crumpet.relative_position_buckets(index, 40)
    grad = torch.randn(3, 64, 33, device="cuda")
    want = crumpet.relative_position_bias_backward(grad, plan)
    long = crumpet.relative_position_buckets(torch.zeros_like(index), 2)
    assert len(long.multi)

    def run(plan, field, at, value):
        t = getattr(plan, field).clone()
        t[at] = value
        crumpet.device_status(clear=True)
        res = crumpet.relative_position_bias_backward(grad, plan._replace(**{field: t}))
        assert crumpet.device_status(clear=True) == 2
        return res

    place = int(plan.order[0])
    got = run(plan, "order", 0, 64 * 33)
    assert torch.equal(got[1:], want[1:])
    left = index.new_tensor(place)
    less = grad.view(3, -1).clone()
    less[:, left] = 0
    assert torch.equal(got, crumpet.relative_position_bias_backward(less.view_as(grad), plan))
    run(plan, "order", 7, -1)
    for at, value in (((39, 0), 40), ((39, 0), -1), ((2, 1), -5), ((39, 2), 64 * 33 + 1)):
        got = run(plan, "items", at, value)
        rows = torch.arange(40, device="cuda") != at[0]
        assert torch.equal(got[rows], want[rows])
    for at, value in (((0, 0), 2), ((0, 0), -1), ((0, 1), -1), ((0, 2), len(long.items) + 1)):
        run(long, "multi", at, value)
    with pytest.raises(ValueError, match="triples"):
        crumpet.relative_position_bias_backward(grad, plan._replace(items=plan.items.view(-1)))
    qkv = torch.randn(1, 64, 3, 3, 16, device="cuda")
    square = crumpet.relative_position_buckets(index[:, :1].expand(64, 64), 40)
    with pytest.raises(ValueError, match="order"):
        crumpet.swin_window_attention_backward(
            torch.randn(1, 64, 48, device="cuda"), qkv, torch.randn(40, 3, device="cuda"),
            square._replace(order=square.order[:-1]))


@pytest.mark.parametrize("length", [20, 50, 100, 300])
def test_bias_gradient_at_the_last_of_2_31_pairs(length):
    """Items at the end of as many pairs as an int counts (13 GB)."""
    n = 2 ** 31 - 1
    order = torch.zeros(n, dtype=torch.int32, device="cuda")
    grad = torch.zeros(1, 1, n, dtype=F16, device="cuda")
    grad[0, 0, 0] = 1
    order[-1], grad[0, 0, -1] = n - 1, 3
    plan = training.RelativePositionBuckets(
        index=None, pairs=torch.zeros((1, 1), dtype=torch.int32, device="cuda").expand(1, n),
        order=order, items=torch.tensor([[0, n - length, n]], dtype=torch.int32, device="cuda"),
        multi=torch.zeros((0, 3), dtype=torch.int32, device="cuda"), num_buckets=1)
    crumpet.device_status(clear=True)
    got = crumpet.relative_position_bias_backward(grad, plan)
    assert float(got) == length + 2 and crumpet.device_status(clear=True) == 0


def test_tangents_are_refused():
    """Through the functions, from tensors that need no gradient (a result without its tangent
    would be a derivative of zero); without tangents the ops record nothing, as before."""
    from test_training_edges import dual_calls

    x = torch.randn(4, 32, device="cuda")
    index = torch.zeros((8, 8), dtype=torch.long, device="cuda")
    plan = crumpet.relative_position_buckets(index, 1)
    table = torch.randn(1, 2, device="cuda")
    qkv = torch.randn(1, 8, 3, 2, 16, device="cuda")
    for f, args in ((crumpet.gelu_checkpoint, (x,)),
                    (lambda t: crumpet.relative_position_bias(t, plan), (table,)),
                    (lambda q: crumpet.swin_window_attention_train(q, table, plan), (qkv,)),
                    (lambda t: crumpet.swin_window_attention_train(qkv, t, plan), (table,)),
                    (lambda b: crumpet.norm_gate_residual(b, x)[0], (x,)),
                    (lambda w: crumpet.norm_gate_residual(x, x, pre_norm=(w, w))[1], (x[0],)),
                    (lambda b: crumpet.checkpointed_mlp(b, x, None, x.t(), None), (x,))):
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(f, args, tuple(map(torch.ones_like, args)))
        with torch.autograd.forward_ad.dual_level():
            duals = tuple(torch.autograd.forward_ad.make_dual(a, torch.ones_like(a)) for a in args)
            with pytest.raises((NotImplementedError, RuntimeError)):
                f(*duals)
    with torch.autograd.forward_ad.dual_level():
        for call in dual_calls("cuda"):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    leaf = x.clone().requires_grad_(True)
    y, kept, scales = torch.ops.crumpet_ops.gelu_checkpoint(leaf)
    assert not y.requires_grad and torch.equal(y, crumpet.gelu_checkpoint(x)[0])


@pytest.mark.parametrize("c", [64, 50])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_gelu_checkpoint_of_the_largest_values(dtype, c):
    """What is finite reads back finite, within a step (and half a step below the top binade's
    last step, as everywhere)."""
    top = torch.finfo(dtype).max
    scale = 2.0 ** (10 if dtype == F16 else 122)
    below = [top, 63.75 * scale, 63.5 * scale, 63.25 * scale, 62.75 * scale, 63.5 * scale / 32]
    x = torch.zeros(2 * len(below), c, dtype=dtype, device="cuda")
    for i, v in enumerate(below):
        x[i, 3], x[i, 7], x[i, 35] = v, -v / 2, -v
        x[i + len(below), 3] = -v
    y, kept = crumpet.gelu_checkpoint(x)
    back = crumpet.restore_activation(kept)
    # (on the CPU: powers of two are exact there)
    step = (2.0 ** (kept.scales.double().cpu() - 127)).cuda().repeat_interleave(32, 1)[:, :c]
    want = torch.round(x.double() / step)
    tops = kept.scales.repeat_interleave(32, 1)[:, :c] == (137 if dtype == F16 else 249)
    assert tops.any()
    want = torch.where(tops, want.clamp(-63, 63), want)
    assert torch.equal(kept.kept.double(), want)
    assert torch.equal(back.double(), want * step)
    grad_x, again = crumpet.gelu_checkpoint_backward(torch.ones_like(x), kept)
    for t in (back, again, grad_x, y):
        assert torch.isfinite(t).all()
    assert torch.equal(again, back.clamp(min=0)) and torch.equal(y, x.clamp(min=0))


@pytest.mark.parametrize("dtype,d", [(F32, 16), (F32, 64), (BF16, 128)], ids=str)
def test_attention_from_two_threads(dtype, d):
    """Windows of two sizes, whose kernels take different amounts of shared memory, from two host
    threads on streams of their own."""
    import threading

    cases = [attention_case(win, (1, 1, 1), (0, 0, 0), 1, 1, d, dtype, F32)
             for win in ((6, 6, 6), (5, 5, 7))]
    want = [attention_both(c) for c in cases]
    torch.cuda.synchronize()
    failed = []

    def work(c, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
                for _ in range(400):
                    out = crumpet.swin_window_attention_train(c["qkv"], c["table"], buckets,
                                                              **c["place"])
                    got = (out, *crumpet.swin_window_attention_backward(
                        c["grad"], c["qkv"], c["table"], buckets, **c["place"]))
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, w))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_a_plan_is_ready_for_any_stream():
    """Nothing of it is still to be computed when it is returned (64 M pairs: the last steps take
    the device longer than the host)."""
    index = torch.randint(0, 100, (8192, 8192), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan = crumpet.relative_position_buckets(index, 100)
        assert side.query()
    assert torch.equal(plan.pairs, index.int())


@pytest.mark.parametrize("pre", [True, False])
def test_norm_gate_backward_allocates_its_results(pre):
    """Without gate and post-norm the branch is not kept, and nothing of its size stands in for it."""
    rows, c = 1 << 16, 64
    branch = torch.randn(rows, c, device="cuda", dtype=BF16, requires_grad=True)
    stream = torch.randn(rows, c, device="cuda", requires_grad=True)
    norm = (torch.ones(c, device="cuda"), torch.zeros(c, device="cuda"))
    out, normed = crumpet.norm_gate_residual(branch, stream, pre_norm=norm if pre else None)
    ends = (out, normed) if pre else (out,)
    grads = [torch.randn_like(t) for t in ends]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(ends, (branch, stream), grads)
    torch.cuda.synchronize()
    # the two results, and the partial column sums (at most two CTAs for each of 148 SMs)
    most = rows * c * (2 + 4) + (2 * 148 * 5 * c * 4 if pre else 0) + (1 << 14)
    assert torch.cuda.max_memory_allocated() - before <= most
    if not pre:
        assert torch.equal(got[1], grads[0]) and torch.equal(got[0], grads[0].to(BF16))


@pytest.mark.parametrize("size", [14, 20])
def test_stage_without_8_bit_activations(size):
    """In fp32 the stage's gradients then have fp32 errors: 1e-5 per operator (as above), some ten
    of them in a row in two blocks."""
    from crumpet_b200 import swin_unetr
    from test_training_gpu import _grads

    torch.manual_seed(3)
    make = lambda: swin_unetr.BasicLayer(48, 2, 3, (7, 7, 7),  # noqa: E731
                                         downsample=swin_unetr.PatchMerging).cuda()
    layer, wide = make(), make()
    wide.load_state_dict(layer.state_dict())
    x = torch.randn(1, 48, size, size, size - 1, device="cuda")
    want_out, want = _grads(wide.double(), x.double(), None)
    assert crumpet.enable_training_kernels(layer, eight_bit_activations=False) == 1
    out, got = _grads(layer.train(), x, None)
    assert rel(out, want_out) <= 1e-4
    for name, w in want.items():
        assert rel(got[name], w) <= 1e-4, name


@pytest.mark.parametrize("off", ["-inf", "lowest", "-1e9"])
@pytest.mark.parametrize("d", [16, 32, 64])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_buckets_switched_off(dtype, d, off):
    """A bucket whose bias excludes its pairs: they weigh nothing, in both directions, and the
    pairs beside them are as before."""
    c = attention_case((3, 4, 5), (2, 1, 2), (1, 0, 2), 1, 2, d, dtype, F32)
    value = {"-inf": -float("inf"), "lowest": torch.finfo(F32).min, "-1e9": -1e9}[off]
    c["table"][::4] = value
    c["table"][c["table"].shape[0] // 2] = 0.25  # a token and itself
    want = attention_wide(dict(c, table=c["table"].clamp(min=-1e30)))
    got = attention_both(c)
    for a, b, tol in zip(got, want, (1.5 * TOL[dtype], TOL[dtype], TOL[F32])):
        assert torch.isfinite(a.float()).all()
        assert rel(a, b) <= tol
    assert not got[2][:4:4].any()


@pytest.mark.parametrize("shift", [-1e4, 1e4])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_bias_of_one_value(dtype, shift):
    """A bias that is the same for all pairs changes nothing, however low (27 tokens: padded
    keys do not take over).  Scores of 4e4 over the scale lose 2^-9 each in fp32, 1e-3 of p."""
    c = attention_case((3, 3, 3), (2, 2, 2), (1, 1, 1), 1, 2, 16, dtype, F32)
    c["table"].fill_(shift)
    got, want = attention_both(c), attention_wide(c)
    for a, b, tol in zip(got[:2], want, (1.5 * TOL[dtype], TOL[dtype])):
        assert torch.isfinite(a.float()).all()
        assert rel(a, b) <= tol + 2e-3


def test_gelu_tails():
    """Formula 7.1.26 bounds erf's error by 1.5e-7 absolutely, so gelu(x) = x F(x) is off by at most
    0.75e-7 |x| in all of the tail (and the hardware's exponential and reciprocal, and fp32
    rounding, by 2^-20 of the value), though not by a part of the value itself."""
    x = torch.linspace(-14, 14, 1 << 16, device="cuda").view(-1, 32)
    y, _ = crumpet.gelu_checkpoint(x)
    want = torch.nn.functional.gelu(x.double())
    off = (y.double() - want).abs()
    assert (off <= 0.75e-7 * x.double().abs() + 2.0 ** -20 * want.abs()).all()
    assert (y[x < -13.5] == 0).all() and torch.equal(y[x > 6], x[x > 6])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_inference_attention_small_scale(dtype):
    """The inference functions follow the same rule, with and without prebuilt tiles."""
    c = attention_case((3, 3, 3), (2, 2, 2), (1, 1, 1), 1, 2, 16, dtype, F32)
    c["qkv"][:, :, :2] *= 16
    c["scale"] = scale = 1e-3
    want = attention_wide(c)[0]
    tiles = fused_attention.attention_bias_tiles(c["table"], c["index"], 27, scale, dtype)
    for t in (None, tiles):
        got = crumpet.swin_window_attention_qkv(c["qkv"], c["table"], c["index"], **c["place"],
                                                scale=scale, bias_tiles=t)
        assert rel(got, want) <= 1.5 * TOL[dtype]
    with pytest.raises(RuntimeError, match="scale"):
        torch.ops.crumpet_ops.swin_window_attention_qkv_tiles(
            torch.empty_like(got), c["qkv"], tiles, [2, 2, 2], [3, 3, 3], [1, 1, 1], scale)
