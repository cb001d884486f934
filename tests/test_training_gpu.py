"""Training operators (crumpet_b200.training) against plain 64-bit implementations.

Tolerances are relative errors in the 2-norm.  An output of p significant bits is rounded to
nearest, an error of at most u = 2^-p per element; where a kernel also rounds one factor of a
long product (P or dS of the attention), those errors are independent and add up like one more
rounding, so 2 u covers both (measured in the norm, well below the worst case per element).
fp32 results: a sum of K products carries at most K 2^-24 of its terms' magnitudes and about
sqrt(K) 2^-24 in the norm; K is at most a few thousand here, so 64 * 2^-24 = 4e-6, and 1e-5
leaves room for the hardware exponential (2^-22) in the softmax.
"""

from __future__ import annotations

import math

import pytest
import torch

import crumpet_b200 as crumpet
from crumpet_b200 import _ops
from crumpet_b200.training import GROUP

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 1e-5, F16: 2 * 2.0 ** -11, BF16: 2 * 2.0 ** -8}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    assert a.shape == b.shape
    n = b.norm()
    return float((a - b).norm() / n) if n > 0 else float((a - b).norm())


def close(a, b, tol=None):
    assert torch.isfinite(a.float()).all()
    assert rel(a, b) <= (TOL[a.dtype] if tol is None else tol)


def window_index(win, device="cuda"):
    c = torch.stack(torch.meshgrid(*(torch.arange(w) for w in win), indexing="ij")).flatten(1)
    r = c[:, :, None] - c[:, None, :] + (torch.tensor(win) - 1)[:, None, None]
    return ((r[0] * (2 * win[1] - 1) + r[1]) * (2 * win[2] - 1) + r[2]).to(device)


def dense_mask(grid, win, shift):
    """The shifted-window mask by MONAI's construction (the package's eager reference)."""
    dims = [g * w for g, w in zip(grid, win)]
    return crumpet.compute_attn_mask_3d_reference(*dims, tuple(win), tuple(shift), torch.float64,
                                                  "cuda")


def attention64(qkv, table, index, mask, scale):
    b, n, _, h, d = qkv.shape
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    s = q @ k.transpose(-1, -2) * scale + table[index].permute(2, 0, 1)
    if mask is not None:
        s = (s.view(-1, mask.shape[0], h, n, n) + mask[:, None]).view(b, h, n, n)
    return (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(b, n, h * d)


def attention_case(win, grid, shift, batch, heads, d, dtype, table_dtype, seed=0, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = win[0] * win[1] * win[2]
    b = batch * grid[0] * grid[1] * grid[2]
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    t = (2 * win[0] - 1) * (2 * win[1] - 1) * (2 * win[2] - 1)
    qkv = rand(b, n, 3, heads, d).to(dtype)
    return dict(qkv=qkv, table=(rand(t, heads) * 0.5).to(table_dtype), index=window_index(win),
                grad=(rand(b, n, heads * d) * std).to(dtype),
                place=dict(num_windows=grid, window_size=win, shift_size=shift),
                mask=dense_mask(grid, win, shift) if any(shift) else None, scale=d ** -0.5)


def check_attention(c):
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    out = crumpet.swin_window_attention_train(c["qkv"], c["table"], buckets, **c["place"])
    gq, gt = crumpet.swin_window_attention_backward(c["grad"], c["qkv"], c["table"], buckets,
                                                    **c["place"])
    qkv = c["qkv"].double().requires_grad_(True)
    table = c["table"].double().requires_grad_(True)
    want = attention64(qkv, table, c["index"], c["mask"], c["scale"])
    wq, wt = torch.autograd.grad(want, (qkv, table), c["grad"].double())
    assert gq.dtype == c["qkv"].dtype and gt.dtype == c["table"].dtype
    # the forward kernel rounds the bias to its element type too (an error of at most u |bias|
    # in a score, |bias| about 0.5 here): one more u
    close(out, want, TOL[out.dtype] * 1.5)
    for part in range(3):  # dq, dk, dv
        close(gq[:, :, part], wq[:, :, part])
    close(gt, wt)


ATTENTION = [
    # window, grid, shift, batch, heads, head dim
    ((7, 7, 7), (2, 2, 2), (3, 3, 3), 1, 3, 16),    # 343 tokens: ragged rows and columns
    ((7, 7, 7), (1, 2, 1), (0, 0, 0), 2, 2, 32),
    ((6, 6, 6), (1, 1, 1), (0, 0, 0), 2, 5, 16),    # 216
    ((4, 4, 4), (3, 2, 2), (2, 2, 2), 1, 4, 32),    # 64: a full tile
    ((5, 13, 1), (2, 1, 3), (2, 0, 0), 1, 3, 16),   # 65: one token past it
    ((2, 8, 8), (2, 2, 1), (1, 4, 0), 1, 2, 16),    # 128, mixed shift
    ((2, 8, 14), (1, 1, 2), (0, 0, 7), 1, 2, 32),   # 224
    ((9, 5, 5), (1, 2, 2), (0, 2, 2), 1, 1, 16),    # 225
    ((2, 16, 11), (1, 2, 1), (0, 8, 0), 1, 1, 16),  # 352: the largest tensor-core window
    ((3, 3, 3), (1, 1, 1), (0, 0, 0), 1, 1, 16),    # 27: one window, one head
    ((2, 1, 1), (3, 1, 1), (0, 0, 0), 1, 2, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "x".join(map(str, c[0])))
def test_attention_tensor_core(case, dtype):
    check_attention(attention_case(*case, dtype, F32))


@pytest.mark.parametrize("case", ATTENTION[3:6], ids=lambda c: "x".join(map(str, c[0])))
def test_attention_16_bit_table(case):
    check_attention(attention_case(*case, BF16, BF16))


@pytest.mark.parametrize("case,dtype", [
    (((7, 7, 7), (2, 1, 1), (3, 0, 0), 1, 2, 16), F32),
    (((5, 5, 5), (1, 2, 2), (0, 2, 2), 1, 3, 32), F32),
    (((3, 3, 3), (1, 1, 1), (0, 0, 0), 2, 2, 64), F32),
    (((2, 3, 7), (2, 1, 1), (1, 0, 0), 1, 2, 256), F32),
    (((4, 4, 4), (1, 1, 2), (0, 0, 2), 1, 2, 64), BF16),
    (((1, 5, 9), (1, 1, 1), (0, 0, 0), 1, 1, 128), F16),
    (((8, 8, 6), (1, 1, 2), (0, 0, 3), 1, 1, 16), F16),  # 384 tokens
], ids=str)
def test_attention_fp32_kernels(case, dtype):
    check_attention(attention_case(*case, dtype, F32))


# fp32 at head dims 16 and 32 multiplies in split products, each 2^-22 from the fp32 one on
# average (2^-20 at most), like the exponential: the same tolerance
@pytest.mark.parametrize("case", [
    ((1, 3, 5), (8, 8, 8), (0, 1, 2), 2, 3, 16),    # one warp per CTA, two windows per CTA
    ((2, 4, 4), (4, 4, 4), (1, 2, 2), 4, 2, 32),    # 32 tokens: a block
    ((3, 11, 1), (2, 2, 1), (1, 5, 0), 1, 2, 16),   # 33: one past it
    ((7, 7, 7), (1, 2, 2), (0, 3, 3), 1, 2, 32),    # bias by tiles
    ((8, 8, 8), (2, 1, 1), (4, 0, 0), 1, 1, 16),    # 512
], ids=str)
def test_attention_fp32_split_products(case):
    check_attention(attention_case(*case, F32, F32))


@pytest.mark.parametrize("d", [16, 32])
def test_attention_fp32_unaligned(d):
    """Tensors off 16-byte boundaries give the same bits as aligned ones."""
    c = attention_case((3, 5, 5), (2, 1, 1), (1, 0, 0), 1, 2, d, F32, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])

    def off(t):
        return torch.empty(t.numel() + 1, device="cuda")[1:].view(t.shape).copy_(t)

    a = (c["grad"], c["qkv"], c["table"], buckets)
    u = (off(c["grad"]), off(c["qkv"]), c["table"], buckets)
    for x, y in zip(crumpet.swin_window_attention_backward(*a, **c["place"]),
                    crumpet.swin_window_attention_backward(*u, **c["place"])):
        assert torch.equal(x, y)
    assert torch.equal(crumpet.swin_window_attention_train(*a[1:], **c["place"]),
                       crumpet.swin_window_attention_train(*u[1:], **c["place"]))


def test_attention_one_token():
    """A window of one token: softmax of one score; only v has a gradient."""
    for dtype in (F32, BF16):
        c = attention_case((1, 1, 1), (2, 1, 1), (0, 0, 0), 1, 2, 16, dtype, F32)
        buckets = crumpet.relative_position_buckets(c["index"], 1)
        gq, gt = crumpet.swin_window_attention_backward(c["grad"], c["qkv"], c["table"], buckets,
                                                        **c["place"])
        assert torch.equal(gq[:, :, 2].reshape(c["grad"].shape), c["grad"])
        # dp - delta of the only key: rounding of one product of 16 terms
        assert gq[:, :, :2].abs().max() < 1e-4 and gt.abs().max() < 1e-4


def test_attention_fp16_loss_scaled_gradient():
    """Large fp16 gradients, as under loss scaling, do not overflow in ds."""
    check_attention(attention_case((7, 7, 7), (1, 1, 2), (0, 0, 3), 1, 2, 16, F16, F32, std=1e3))


def test_attention_fp16_small_gradients_keep_their_bits():
    """ds of fp16 gradients 2^-12 times as large is 2^-12 times the same bits, although most of
    it is below fp16's least normal number by itself: the table's fp32 gradient scales exactly,
    and grad_qkv up to the storage of either result (fp16 numbers 2^-24 apart at the least)."""
    c = attention_case((7, 7, 7), (1, 1, 2), (0, 0, 3), 1, 2, 16, F16, F32)
    big = (c["grad"] * 8).round() / 8  # multiples of 1/8: exact in fp16 after the scaling too
    small = big * 2.0 ** -12
    assert torch.equal(small.double(), big.double() * 2.0 ** -12)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    run = lambda g: crumpet.swin_window_attention_backward(g, c["qkv"], c["table"], buckets,  # noqa: E731
                                                           **c["place"])
    (bq, bt), (sq, st) = run(big), run(small)
    assert torch.equal(st, bt * 2.0 ** -12)
    want = bq.double() * 2.0 ** -12
    assert ((sq.double() - want).abs() <= 2.0 ** -25 + 2.0 ** -11 * want.abs()).all()


def test_attention_large_scores_and_heavy_mask():
    """Scores over 100 apart: the mask is -100, as in the forward, not an exclusion."""
    c = attention_case((4, 4, 4), (2, 1, 1), (2, 0, 0), 1, 2, 16, F32, F32)
    c["qkv"][:, :, :2] *= 6
    check_attention(c)


def test_attention_results_do_not_change_from_run_to_run():
    c = attention_case((7, 7, 7), (3, 3, 3), (3, 3, 3), 1, 3, 16, BF16, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    args = (c["grad"], c["qkv"], c["table"], buckets)
    first = crumpet.swin_window_attention_backward(*args, **c["place"])
    for _ in range(3):
        again = crumpet.swin_window_attention_backward(*args, **c["place"])
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_attention_autograd_strides_and_stream():
    """Through autograd, from a strided qkv and gradient, on another stream."""
    c = attention_case((4, 4, 4), (2, 2, 1), (2, 2, 0), 1, 2, 16, BF16, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    want = crumpet.swin_window_attention_backward(c["grad"], c["qkv"], c["table"], buckets,
                                                  **c["place"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        wide = torch.stack((c["qkv"], c["qkv"]), -1)[..., 0].detach().requires_grad_(True)
        assert not wide.is_contiguous()
        table = c["table"].clone().requires_grad_(True)
        out = crumpet.swin_window_attention_train(wide, table, buckets, **c["place"])
        got = torch.autograd.grad(out, (wide, table), torch.stack((c["grad"],) * 2, -1)[..., 0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_unaligned_takes_the_fp32_kernels():
    c = attention_case((3, 3, 3), (2, 1, 1), (1, 0, 0), 1, 2, 16, BF16, F32)
    flat = torch.empty(c["qkv"].numel() + 1, dtype=BF16, device="cuda")
    flat[1:] = c["qkv"].reshape(-1)
    c["qkv"] = flat[1:].view(c["qkv"].shape)
    assert c["qkv"].data_ptr() % 16
    check_attention(c)


def test_attention_no_windows():
    c = attention_case((3, 3, 3), (1, 1, 1), (0, 0, 0), 1, 2, 16, BF16, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    gq, gt = crumpet.swin_window_attention_backward(c["grad"][:0], c["qkv"][:0], c["table"], buckets)
    assert gq.numel() == 0 and not gt.any()


def test_attention_gradient_against_differences():
    """Directional derivatives of the kernel's own fp32 forward: central differences at step h
    err by h^2 f'''/6 and by the forward's rounding 2^-24 sqrt(terms) / h, 1e-3 at h = 1e-2."""
    c = attention_case((3, 3, 3), (2, 1, 1), (1, 0, 0), 1, 2, 16, F32, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    gq, gt = crumpet.swin_window_attention_backward(c["grad"], c["qkv"], c["table"], buckets,
                                                    **c["place"])
    f = lambda q, t: float((crumpet.swin_window_attention_train(q, t, buckets, **c["place"])  # noqa: E731
                            .double() * c["grad"].double()).sum())
    h = 1e-2
    for along_table in (False, True):
        d = torch.randn_like(c["table"] if along_table else c["qkv"])
        d /= d.norm()
        q, t = (c["qkv"], c["table"])
        if along_table:
            diff, got = f(q, t + h * d) - f(q, t - h * d), (gt.double() * d).sum()
            size = gt.norm()
        else:
            diff, got = f(q + h * d, t) - f(q - h * d, t), (gq.double() * d).sum()
            size = gq.norm()
        assert abs(diff / (2 * h) - float(got)) <= 1e-3 * float(size)


def test_attention_refusals():
    c = attention_case((3, 3, 3), (2, 1, 1), (1, 0, 0), 1, 2, 16, BF16, F32)
    buckets = crumpet.relative_position_buckets(c["index"], c["table"].shape[0])
    run = crumpet.swin_window_attention_train
    q, t = c["qkv"], c["table"]
    with pytest.raises(ValueError, match="B, N, 3, H"):
        run(q[:, :, :2], t, buckets)
    with pytest.raises(ValueError, match="index"):
        run(q[:, :20], t, buckets)
    with pytest.raises(ValueError, match="table"):
        run(q, t[:, :1], buckets)
    with pytest.raises(ValueError, match="table"):
        run(q, t[:5], buckets)
    with pytest.raises(ValueError, match="window_size"):
        run(q, t, buckets, (2, 1, 1), (3, 3, 2), (0, 0, 0))
    with pytest.raises(ValueError, match="shift"):
        run(q, t, buckets, (2, 1, 1), (3, 3, 3), (3, 0, 0))
    with pytest.raises(ValueError, match="multiple"):
        run(q, t, buckets, (3, 1, 1), (3, 3, 3), (1, 0, 0))
    with pytest.raises(ValueError, match="scale"):
        run(q, t, buckets, scale=float("nan"))
    with pytest.raises(ValueError, match="head_dim"):
        run(q.reshape(2, 27, 3, 4, 8), t[:, :1].expand(-1, 4), buckets)
    with pytest.raises(TypeError):
        run(q.double(), t, buckets)
    with pytest.raises(RuntimeError, match="CUDA"):
        run(q.cpu(), t, buckets)
    with pytest.raises(ValueError, match="grad_out"):
        crumpet.swin_window_attention_backward(c["grad"].float(), q, t, buckets)


# ------------------------------------------------------------------------------ bias
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,buckets,heads", [
    (343, 343, 2197, 3), (1, 1, 1, 1), (1, 77, 5, 24), (130, 9, 64, 2),
    (200, 201, 1, 3),       # one bucket of 40,200 pairs: cut into items and joined
    (64, 64, 20000, 2),     # more buckets than pairs, and than shared memory holds
], ids=str)
def test_bias(rows, cols, buckets, heads, dtype):
    g = torch.Generator("cuda").manual_seed(1)
    index = torch.randint(0, buckets, (rows, cols), generator=g, device="cuda")
    table = torch.randn((buckets, heads), generator=g, device="cuda").to(dtype)
    grad = torch.randn((heads, rows, cols), generator=g, device="cuda").to(dtype)
    plan = crumpet.relative_position_buckets(index, buckets)
    bias = crumpet.relative_position_bias(table, plan)
    assert torch.equal(bias, table[index].permute(2, 0, 1))
    want = torch.zeros((buckets, heads), dtype=torch.float64, device="cuda").index_add_(
        0, index.reshape(-1), grad.double().permute(1, 2, 0).reshape(-1, heads))
    got = crumpet.relative_position_bias_backward(grad, plan)
    assert got.dtype == dtype
    close(got, want)
    assert torch.equal(got, crumpet.relative_position_bias_backward(grad, plan))


def test_bias_autograd_dtypes_and_strides():
    index = window_index((3, 2, 4))
    plan = crumpet.relative_position_buckets(index, 5 * 3 * 7)
    table = torch.randn(105, 3, device="cuda", requires_grad=True)
    bias = crumpet.relative_position_bias(table, plan, torch.bfloat16)
    assert bias.dtype == BF16
    w = torch.randn(24, 3, 24, device="cuda", dtype=BF16).transpose(0, 1)  # a strided gradient
    (got,) = torch.autograd.grad(bias, table, w)
    assert got.dtype == F32
    want = torch.zeros(105, 3, device="cuda", dtype=torch.float64).index_add_(
        0, index.reshape(-1), w.double().permute(1, 2, 0).reshape(-1, 3))
    close(got, want)
    unaligned = torch.randn(105 * 3 + 1, device="cuda")[1:].view(105, 3)
    assert torch.equal(crumpet.relative_position_bias(unaligned, plan),
                       unaligned[index].permute(2, 0, 1))


def test_bias_empty_index():
    plan = crumpet.relative_position_buckets(torch.zeros((0, 4), dtype=torch.long, device="cuda"), 3)
    assert crumpet.relative_position_bias(torch.ones(3, 2, device="cuda"), plan).shape == (2, 0, 4)
    grad = crumpet.relative_position_bias_backward(torch.ones(2, 0, 4, device="cuda"), plan)
    assert grad.shape == (3, 2) and not grad.any()


def test_bias_refusals():
    plan = crumpet.relative_position_buckets(window_index((2, 2, 2)), 27)
    with pytest.raises(ValueError, match="table"):
        crumpet.relative_position_bias(torch.ones(26, 2, device="cuda"), plan)
    with pytest.raises(TypeError):
        crumpet.relative_position_bias(torch.ones(27, 2, device="cuda", dtype=torch.double), plan)
    with pytest.raises(ValueError, match="grad_bias"):
        crumpet.relative_position_bias_backward(torch.ones(2, 8, 9, device="cuda"), plan)
    with pytest.raises(RuntimeError, match="CUDA"):
        crumpet.relative_position_bias(torch.ones(27, 2), plan)


# ------------------------------------------------------------------------------- norms
def norm64(x, p, eps):
    x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * p[0] + p[1]


def norm_gate64(branch, residual, gate, scale, post, pre, eps, stored):
    n = branch if post is None else norm64(branch, post, eps)
    if gate is not None:
        n = n * gate
    if scale is not None:
        n = (n.reshape(scale.numel(), -1) * scale[:, None]).reshape(branch.shape)
    out = residual + n
    # the next norm reads the stored stream: its value, with the sum's gradient
    seen = out + (stored.double() - out).detach()
    return out, None if pre is None else norm64(seen, pre, eps)


def norm_case(rows, c, dtype, stream, post, gate, scale, pre, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    vec = lambda m: rand(c) * 0.2 + m  # noqa: E731
    return dict(branch=rand(rows, c).to(dtype), residual=(rand(rows, c) + 0.3).to(stream),
                gate=vec(0.7) if gate else None,
                row_scale=torch.tensor([0.0, 1.25, 1.25], device="cuda") if scale else None,
                post_norm=(vec(1.0), vec(0.0)) if post else None,
                pre_norm=(vec(1.0), vec(0.0)) if pre else None,
                grad_out=rand(rows, c).to(stream), grad_normed=rand(rows, c).to(dtype))


def check_norm(k, eps=1e-5):
    how = {n: k[n] for n in ("gate", "row_scale", "post_norm", "pre_norm")}
    out, normed = crumpet.norm_gate_residual(k["branch"], k["residual"], eps=eps, **how)
    wide = lambda t: t.double().requires_grad_(True)  # noqa: E731
    branch, residual = wide(k["branch"]), wide(k["residual"])
    gate = None if k["gate"] is None else wide(k["gate"])
    post = None if k["post_norm"] is None else [wide(t) for t in k["post_norm"]]
    pre = None if k["pre_norm"] is None else [wide(t) for t in k["pre_norm"]]
    scale = None if k["row_scale"] is None else k["row_scale"].double()
    w_out, w_normed = norm_gate64(branch, residual, gate, scale, post, pre, eps, out)
    close(out, w_out)
    assert (normed is None) == (pre is None)
    if pre is not None:
        close(normed, w_normed)
    grads = crumpet.norm_gate_residual_backward(
        k["grad_out"], k["grad_normed"] if pre is not None else None, out, k["branch"], eps=eps,
        **how)
    leaves = [residual, branch, gate, *(post or (None, None)), *(pre or (None, None))]
    ends = [w_out] + ([] if pre is None else [w_normed])
    seeds = [k["grad_out"].double()] + ([] if pre is None else [k["grad_normed"].double()])
    want = iter(torch.autograd.grad(ends, [t for t in leaves if t is not None], seeds))
    for leaf, got in zip(leaves, grads):
        assert (leaf is None) == (got is None)
        if leaf is not None:
            close(got, next(want))
    return grads


FLAGS = [(False, False, False, True), (True, True, True, True), (False, True, False, False),
         (True, False, True, True), (False, False, True, False), (True, True, False, False)]


@pytest.mark.parametrize("flags", FLAGS, ids=str)
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (F16, F32), (F32, F32)], ids=str)
@pytest.mark.parametrize("rows,c", [(3 * 343, 48), (3, 768), (39, 100)])
def test_norm_gate(rows, c, dtype, stream, flags):
    check_norm(norm_case(rows, c, dtype, stream, *flags))


@pytest.mark.parametrize("c", [8, 9, 24, 256, 257, 264, 513, 1024, 2040, 2049, 4096])
@pytest.mark.parametrize("dtype,stream", [(BF16, F32), (F16, F16), (F32, F32)], ids=str)
def test_norm_gate_widths(c, dtype, stream):
    check_norm(norm_case(21, c, dtype, stream, True, True, True, True))


def test_norm_gate_many_rows():
    """More rows than one pass of the backward's grid."""
    check_norm(norm_case(3 * 20011, 40, BF16, BF16, True, True, True, True))


def test_norm_gate_row_of_one_value():
    """A constant row has no variance: the norm gives its bias, and eps keeps the gradient finite."""
    k = norm_case(6, 16, F32, F32, True, True, True, True)
    k["branch"][2] = 3.0
    k["branch"][4] = 0.0
    check_norm(k)


def test_norm_gate_one_channel():
    """LayerNorm of a single channel is its bias; the residual's gradient is grad_out."""
    k = norm_case(3, 1, F32, F32, False, False, False, True)
    out, normed = crumpet.norm_gate_residual(k["branch"], k["residual"], pre_norm=k["pre_norm"])
    assert torch.equal(normed, k["pre_norm"][1].expand(3, 1))
    g = crumpet.norm_gate_residual_backward(k["grad_out"], k["grad_normed"], out, k["branch"],
                                            pre_norm=k["pre_norm"])
    assert torch.equal(g.residual, k["grad_out"]) and not g.pre_weight.any()


def test_norm_gate_dropped_sample_and_determinism():
    k = norm_case(3 * 50, 48, BF16, BF16, False, True, True, True)
    a, b = check_norm(k), check_norm(k)
    assert all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)
    assert not a.branch[:50].any()  # the first sample's branch was dropped
    out, _ = crumpet.norm_gate_residual(k["branch"], k["residual"], k["gate"], k["row_scale"])
    assert torch.equal(out[:50], k["residual"][:50])


def test_norm_gate_autograd_5d_and_unaligned():
    """As a block calls it: [B, D, H, W, C], autograd, parameters in another dtype, a strided
    branch, and tensors off 16-byte boundaries."""
    k = norm_case(3 * 60, 24, F16, F32, True, True, True, True)
    shape = (3, 3, 4, 5, 24)
    how = dict(row_scale=k["row_scale"])
    want_out, want_normed = crumpet.norm_gate_residual(
        k["branch"], k["residual"], k["gate"], k["row_scale"], k["post_norm"], k["pre_norm"])
    want = crumpet.norm_gate_residual_backward(
        k["grad_out"], k["grad_normed"], want_out, k["branch"], k["gate"], k["row_scale"],
        k["post_norm"], k["pre_norm"])
    off = torch.empty(k["residual"].numel() + 1, device="cuda")
    off[1:] = k["residual"].reshape(-1)
    residual = off[1:].view(shape).requires_grad_(True)
    branch = k["branch"].view(shape).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    gate = k["gate"].double().requires_grad_(True)
    post = tuple(t.clone().requires_grad_(True) for t in k["post_norm"])
    pre = tuple(t.clone().requires_grad_(True) for t in k["pre_norm"])
    out, normed = crumpet.norm_gate_residual(branch, residual, gate, post_norm=post, pre_norm=pre,
                                             **how)
    close(out.view(-1, 24), want_out.double())
    close(normed.view(-1, 24), want_normed.double())
    got = torch.autograd.grad((out, normed), (residual, branch, gate, *post, *pre),
                              (k["grad_out"].view(shape), k["grad_normed"].view(shape)))
    assert got[2].dtype == torch.double
    for g, w in zip(got, want):
        close(g.reshape(w.shape).to(w.dtype), w.double())


def test_norm_gate_no_rows():
    k = norm_case(3, 16, BF16, BF16, True, True, False, True)
    empty = {n: k[n][:0] for n in ("branch", "residual", "grad_out", "grad_normed")}
    how = {n: k[n] for n in ("gate", "post_norm", "pre_norm")}
    out, normed = crumpet.norm_gate_residual(empty["branch"], empty["residual"], **how)
    assert out.shape == normed.shape == (0, 16)
    g = crumpet.norm_gate_residual_backward(empty["grad_out"], empty["grad_normed"], out,
                                            empty["branch"], **how)
    assert not any(t.any() for t in g)


def test_norm_gate_refusals():
    k = norm_case(6, 16, BF16, BF16, True, True, False, True)
    f, b, r = crumpet.norm_gate_residual, k["branch"], k["residual"]
    with pytest.raises(ValueError, match="shape"):
        f(b, r[:5])
    with pytest.raises(TypeError):
        f(b, r.half())
    with pytest.raises(ValueError, match="eps"):
        f(b, r, eps=0.0)
    with pytest.raises(ValueError, match="row_scale"):
        f(b, r, row_scale=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="gate"):
        f(b, r, gate=torch.ones(15, device="cuda"))
    with pytest.raises(ValueError, match="pre_norm"):
        f(b, r, pre_norm=(torch.ones(16, device="cuda"),))
    with pytest.raises(ValueError, match="channels"):
        f(torch.zeros(1, 4097, device="cuda"), torch.zeros(1, 4097, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(b.cpu(), r.cpu())
    with pytest.raises(ValueError, match="grad_normed"):
        crumpet.norm_gate_residual_backward(k["grad_out"], None, r, b, pre_norm=k["pre_norm"])


# ------------------------------------------------------------------- 8-bit checkpoints
def eight_bits64(x):
    """By the definition, in 64 bits: the least power of two that reaches the largest value.
    On the CPU, whose powers of two are exact."""
    rows, c = x.shape
    g = torch.nn.functional.pad(x.double().cpu(), (0, -c % GROUP)).view(rows, -1, GROUP)
    top = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 127)).clamp(min=-126)
    e = torch.where(top > 0, e, torch.full_like(e, -126))
    e = torch.where(127 * 2.0 ** (e - 1) >= top, (e - 1).clamp(min=-126), e)  # log2's rounding
    return (torch.round(g / 2.0 ** e) * 2.0 ** e).view(rows, -1)[:, :c].to(x.device)


GELU = [(343, 192), (5, 32), (7, 250), (1, 1), (3, 8), (2, 1537), (64, 40)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,c", GELU)
def test_gelu_checkpoint(rows, c, dtype):
    g = torch.Generator("cuda").manual_seed(rows + c)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = (rand(rows, c) * torch.exp(2 * rand(rows, 1))).to(dtype)  # rows of different sizes
    grad = rand(rows, c).to(dtype)
    y, kept = crumpet.gelu_checkpoint(x)
    assert kept.kept.dtype == torch.int8 and kept.scales.shape == (rows, -(-c // GROUP))
    close(y, torch.nn.functional.gelu(x.double()))
    u = eight_bits64(x)
    # exact: at most 8 bits, which every dtype holds
    assert torch.equal(crumpet.restore_activation(kept).double(), u)
    grad_x, again = crumpet.gelu_checkpoint_backward(grad, kept)
    leaf = u.clone().requires_grad_(True)
    want = torch.nn.functional.gelu(leaf)
    close(again, want)
    close(grad_x, torch.autograd.grad(want, leaf, grad.double())[0])
    # half a step of a group: at most 2^-1 * 2^(1 - 7) of its largest value
    step = (2.0 ** (kept.scales.double().cpu() - 127)).cuda()
    assert ((u - x.double()).abs() <= step.repeat_interleave(GROUP, 1)[:, :c] / 2).all()


def test_gelu_checkpoint_thresholds_and_extremes():
    """Scales at and around 127 times a power of two, zeros, subnormals and the largest values."""
    tops = [127.0, 127.00001, 126.99999, 128.0, 1.0, 0.0, 2.0 ** -140, 2.0 ** -126, 3e38, 254.0]
    x = torch.zeros(len(tops), 64, device="cuda")
    for i, t in enumerate(tops):
        x[i, 3] = -t
        x[i, 40] = t / 3
    _, kept = crumpet.gelu_checkpoint(x)
    assert torch.equal(crumpet.restore_activation(kept).double(), eight_bits64(x))
    assert kept.scales[0, 0] == 127 and kept.scales[1, 0] == 128 and kept.scales[2, 0] == 127


@pytest.mark.parametrize("c", [64, 50])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_gelu_checkpoint_overflow_reads_back_as_nan(bad, c):
    x = torch.randn(3, c, device="cuda", dtype=F16)
    x[1, 5] = bad
    _, kept = crumpet.gelu_checkpoint(x)
    back = crumpet.restore_activation(kept)
    hit = torch.zeros(3, c, dtype=torch.bool, device="cuda")
    hit[1, :32] = True
    assert torch.equal(back.isnan(), hit)
    grad_x, again = crumpet.gelu_checkpoint_backward(torch.ones_like(x), kept)
    assert torch.equal(grad_x.isnan(), hit) and torch.equal(again.isnan(), hit)


def test_gelu_of_infinities():
    """The limits: inf and 0 (torch's product gives NaN for -inf); NaN stays NaN."""
    inf, nan = float("inf"), float("nan")
    for c in (32, 31):
        x = torch.zeros(1, c, device="cuda")
        x[0, :3] = torch.tensor([inf, -inf, nan])
        y, _ = crumpet.gelu_checkpoint(x)
        assert y[0, 0] == inf and y[0, 1] == 0 and y[0, 2].isnan() and not y[0, 3:].any()


def test_gelu_checkpoint_against_differences():
    """grad_x is the slope of gelu at the kept input: differences in 64 bits at 2^-10, an error
    of h^2 f'''/6 below 1e-6."""
    x = torch.linspace(-9, 9, 4096, device="cuda").view(-1, 32)
    _, kept = crumpet.gelu_checkpoint(x)
    u = crumpet.restore_activation(kept).double()
    f, h = torch.nn.functional.gelu, 2.0 ** -10
    slope = (f(u + h) - f(u - h)) / (2 * h)
    grad_x, _ = crumpet.gelu_checkpoint_backward(torch.ones_like(x), kept)
    assert (grad_x.double() - slope).abs().max() < 2e-6


def test_gelu_checkpoint_strides_unaligned_and_empty():
    x = torch.randn(65, 33, device="cuda", dtype=BF16).t()
    y, kept = crumpet.gelu_checkpoint(x)
    y2, kept2 = crumpet.gelu_checkpoint(x.contiguous())
    assert torch.equal(y, y2) and torch.equal(kept.kept, kept2.kept)
    flat = torch.randn(4 * 64 + 1, device="cuda", dtype=BF16)
    a = flat[1:].view(4, 64)
    y, kept = crumpet.gelu_checkpoint(a)
    y2, kept2 = crumpet.gelu_checkpoint(a.clone())
    assert torch.equal(kept.kept, kept2.kept) and torch.equal(kept.scales, kept2.scales)
    assert torch.equal(y, y2)
    for shape in ((0, 64), (3, 0)):
        y, kept = crumpet.gelu_checkpoint(torch.empty(shape, device="cuda"))
        gx, again = crumpet.gelu_checkpoint_backward(torch.empty(shape, device="cuda"), kept)
        assert y.shape == gx.shape == again.shape == shape


def test_gelu_checkpoint_refusals():
    x = torch.randn(2, 32, device="cuda")
    with pytest.raises(TypeError):
        crumpet.gelu_checkpoint(x.double())
    with pytest.raises(RuntimeError, match="CUDA"):
        crumpet.gelu_checkpoint(x.cpu())
    with pytest.raises(RuntimeError, match="checkpointed_mlp"):
        crumpet.gelu_checkpoint(x.requires_grad_(True))
    _, kept = crumpet.gelu_checkpoint(x.detach())
    with pytest.raises(ValueError, match="grad_y"):
        crumpet.gelu_checkpoint_backward(torch.zeros(2, 31, device="cuda"), kept)
    with pytest.raises(ValueError, match="grad_y"):
        crumpet.gelu_checkpoint_backward(torch.zeros(2, 32, device="cuda", dtype=F16), kept)


def test_checkpointed_mlp():
    """Forward as the eager MLP's; gradients as its formulas give them for the kept activation."""
    g = torch.Generator("cuda").manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = rand(2, 5, 48).requires_grad_(True)
    w1, b1, w2, b2 = (t.requires_grad_(True) for t in (rand(192, 48) * 0.1, rand(192) * 0.1,
                                                      rand(48, 192) * 0.1, rand(48) * 0.1))
    grad = rand(2, 5, 48)
    out = crumpet.checkpointed_mlp(x, w1, b1, w2, b2)
    got = torch.autograd.grad(out, (x, w1, b1, w2, b2), grad)
    wide = [t.detach().double() for t in (x, w1, b1, w2, b2)]
    u = wide[0] @ wide[1].t() + wide[2]
    close(out, torch.nn.functional.gelu(u) @ wide[3].t() + wide[4])
    # the kernel's own fp32 u, quantised by the definition
    u32 = torch.nn.functional.linear(x.detach(), w1.detach(), b1.detach())
    k = eight_bits64(u32.view(-1, 192)).requires_grad_(True)
    y = torch.nn.functional.gelu(k)
    go = grad.double().view(-1, 48)
    (gu,) = torch.autograd.grad(y, k, go @ wide[3])
    want = ((gu @ wide[1]).view(x.shape), gu.t() @ wide[0].view(-1, 48), gu.sum(0),
            go.t() @ y.detach(), go.sum(0))
    for a, b in zip(got, want):
        close(a, b)
    for amp in (F16, BF16):
        with torch.autocast("cuda", amp):
            o = crumpet.checkpointed_mlp(x, w1, None, w2, b2)
            assert o.dtype == amp
        (gx,) = torch.autograd.grad(o, x, grad.to(amp))
        assert gx.dtype == F32 and torch.isfinite(gx).all()


# --------------------------------------------------------------- the training path together
def _grads(model, x, amp):
    for p in model.parameters():
        p.grad = None
    with torch.autocast("cuda", amp, enabled=amp is not None):
        out = model(x)
        loss = (out.float() ** 2).mean()
    loss.backward()
    return out.detach(), {n: p.grad.detach().clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("size", [14, 20, 6])
@pytest.mark.parametrize("amp", [None, BF16], ids=str)
def test_stage_trains_as_the_eager_one(size, amp):
    """A stage (shifted and unshifted block, patch merging) with the training kernels against
    the eager stage in 64 bits: volumes that are, are not and are smaller than window
    multiples.  The hidden activation's 8 bits (steps of 2^-7 of a group's largest value, a
    relative error of about 2^-8 / sqrt 3 in it) bound the weight gradients, 16-bit matrix
    products the rest: 2e-2 without, 6e-2 with autocast."""
    from crumpet_b200 import swin_unetr

    torch.manual_seed(3)
    layer = swin_unetr.BasicLayer(48, 2, 3, (7, 7, 7), downsample=swin_unetr.PatchMerging).cuda()
    x = torch.randn(2, 48, size, size, size - 1 if size > 7 else size, device="cuda")
    wide = swin_unetr.BasicLayer(48, 2, 3, (7, 7, 7), downsample=swin_unetr.PatchMerging).cuda()
    wide.load_state_dict(layer.state_dict())
    want_out, want = _grads(wide.double(), x.double(), None)
    assert crumpet.enable_training_kernels(layer) == 1
    layer.train()
    from crumpet_b200 import profiling

    before = profiling.counters["swin_window_attention_backward"]
    out, got = _grads(layer, x, amp)
    assert profiling.counters["swin_window_attention_backward"] == before + 2
    tol = 2e-2 if amp is None else 6e-2
    assert rel(out, want_out) <= (1e-4 if amp is None else 2e-2)
    for name, w in want.items():
        assert rel(got[name], w) <= tol, name
    # eval mode and disabling give the layer's own forward back
    layer.eval()
    with torch.no_grad():
        own = type(layer).forward(layer, x)
        assert torch.equal(layer(x), own)
    assert crumpet.disable_training_kernels(layer) == 1
    assert "forward" not in layer.__dict__


def test_stage_with_dropout_keeps_its_own_forward():
    from crumpet_b200 import profiling, swin_unetr

    layer = swin_unetr.BasicLayer(48, 1, 3, (7, 7, 7), attn_drop=0.1).cuda().train()
    crumpet.enable_training_kernels(layer)
    before = profiling.total_launches()
    layer(torch.randn(1, 48, 7, 7, 7, device="cuda"))
    assert profiling.total_launches() == before


def test_stage_drop_path():
    """A dropped sample passes through its blocks unchanged; the others' branches scale by
    1 / keep."""
    from crumpet_b200 import swin_unetr

    class DropPath(torch.nn.Module):
        drop_prob, scale_by_keep = 0.5, True

    layer = swin_unetr.BasicLayer(48, 1, 3, (7, 7, 7)).cuda().train()
    layer.blocks[0].drop_path = DropPath()
    crumpet.enable_training_kernels(layer)
    x = torch.randn(16, 48, 7, 7, 7, device="cuda")
    same = [(layer(x) - x).abs().amax((1, 2, 3, 4)) for _ in range(4)]
    dropped = torch.stack(same) == 0
    assert dropped.any() and not dropped.all()


def test_whole_model_trains():
    """One optimiser step of the bundled network with the training kernels lowers the loss on
    its own batch, and no kernel reports an error."""
    from crumpet_b200 import swin_unetr

    torch.manual_seed(0)
    model = swin_unetr.SwinUNETR(1, 4, 48).cuda().train()
    assert crumpet.enable_training_kernels(model) == 4
    opt = torch.optim.SGD(model.parameters(), lr=1e-2)
    x = torch.randn(1, 1, 64, 64, 64, device="cuda")
    target = torch.randint(0, 4, (1, 64, 64, 64), device="cuda")
    losses = []
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast("cuda", BF16):
            loss = torch.nn.functional.cross_entropy(model(x).float(), target)
        loss.backward()
        assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)
        opt.step()
        losses.append(float(loss))
    assert losses[-1] < losses[0] and math.isfinite(losses[-1])
    assert crumpet.device_status() == 0


def test_traced_shapes(monkeypatch):
    """What tracing is told about each op's results is what the op returns."""
    from crumpet_b200 import training

    seen, launch = {}, training._launch

    def record(name, work, *args):
        res = launch(name, work, *args)
        same = lambda t: [(r.shape, r.dtype) for r in (t if isinstance(t, (tuple, list)) else [t])]  # noqa: E731
        assert same(training.FAKE_IMPLS[name](*args)) == same(res), name
        seen[name] = True
        return res

    monkeypatch.setattr(training, "_launch", record)
    w = torch.ones(48, device="cuda", dtype=F16)
    x = torch.randn(6, 48, device="cuda", dtype=F16)
    out, normed = crumpet.norm_gate_residual(x, x.float(), w, None, (w, w), (w, w))
    crumpet.norm_gate_residual(x, x)
    crumpet.norm_gate_residual_backward(out, normed, out, x, w, None, (w, w), (w, w))
    crumpet.norm_gate_residual_backward(out, None, out, x)
    y, kept = crumpet.gelu_checkpoint(x)
    crumpet.gelu_checkpoint_backward(y, kept)
    crumpet.restore_activation(kept)
    b = crumpet.relative_position_buckets(window_index((2, 2, 2)), 27)
    table = torch.randn(27, 3, device="cuda")
    crumpet.relative_position_bias_backward(crumpet.relative_position_bias(table, b, BF16), b, F16)
    qkv = torch.randn(2, 8, 3, 3, 16, device="cuda", dtype=F16)
    place = (table, b, (1, 1, 1), (2, 2, 2))
    o = crumpet.swin_window_attention_train(qkv, *place)
    crumpet.swin_window_attention_backward(o, qkv, *place)
    assert set(seen) == set(training.FAKE_IMPLS)


# -------------------------------------------------------------------------------- C ABI
def test_second_derivatives_are_refused():
    """The gradients are not differentiable again: asked for, that is an error, not a wrong sum."""
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    table = torch.randn(27, 2, device="cuda", requires_grad=True)
    qkv = torch.randn(1, 8, 3, 2, 16, device="cuda", requires_grad=True)
    b = crumpet.relative_position_buckets(window_index((2, 2, 2)), 27)
    w = torch.ones(32, device="cuda")
    weight = torch.randn(32, 32, device="cuda", requires_grad=True)
    for out, wrt in (
            (crumpet.relative_position_bias(table, b), table),
            (crumpet.swin_window_attention_train(qkv, table, b, window_size=(2, 2, 2)), qkv),
            (crumpet.norm_gate_residual(x, x, pre_norm=(w, w))[1], x),
            (crumpet.checkpointed_mlp(x, weight, None, weight, None), x)):
        g, = torch.autograd.grad((out ** 2).sum(), wrt, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad((g ** 2).sum(), wrt)


def test_c_abi():
    """The entry points called directly give what the Python functions give."""
    import ctypes

    from helpers import ptr, stream_ptr

    lib = _ops.capi()
    x = torch.randn(7, 48, device="cuda", dtype=BF16)
    y, kept = torch.empty_like(x), torch.empty(7, 48, dtype=torch.int8, device="cuda")
    scales = torch.empty(7, 2, dtype=torch.uint8, device="cuda")
    assert lib.crumpet_gelu_checkpoint(ptr(y), ptr(kept), ptr(scales), ptr(x), 2, 7, 48,
                                       stream_ptr()) == 0
    wy, w = crumpet.gelu_checkpoint(x)
    assert torch.equal(y, wy) and torch.equal(kept, w.kept) and torch.equal(scales, w.scales)
    out = torch.empty_like(x)
    null = ctypes.c_void_p(0)
    assert lib.crumpet_norm_gate_residual(ptr(out), null, ptr(x), ptr(y), 2, 2, null, null, 1, null,
                                          null, null, null, 1e-5, 7, 48, stream_ptr()) == 0
    assert torch.equal(out, (x.float() + y.float()).to(BF16))
