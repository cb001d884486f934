"""Training operators: what needs no GPU -- the bucket plan, refusals, meta shapes, the C ABI's
argument checks and the switch on a model."""

from __future__ import annotations

import ctypes

import pytest
import torch

import crumpet_b200 as crumpet
from crumpet_b200 import _ops, swin_unetr, training


def _check_plan(index, buckets):
    plan = crumpet.relative_position_buckets(index, buckets)
    flat = index.reshape(-1)
    seen = torch.zeros(buckets, dtype=torch.bool)
    at = 0
    several = {int(b): (int(f), int(e)) for b, f, e in plan.multi}
    owner = {i: b for b, (f, e) in several.items() for i in range(f, e)}
    for i, (bucket, begin, end) in enumerate(plan.items.tolist()):
        assert (bucket == -1) == (i in owner)
        bucket = owner.get(i, bucket)
        seen[bucket] = True
        assert begin == at and 0 <= end - begin <= training._ITEM
        at = end
        assert (flat[plan.order[begin:end].long()] == bucket).all()
    assert at == flat.numel() and seen.all()
    assert sorted(plan.order.tolist()) == list(range(flat.numel()))
    for _, (first, last) in several.items():
        assert last - first > 1
    return plan


def test_bucket_plan():
    g = torch.Generator().manual_seed(0)
    _check_plan(torch.randint(0, 7, (31, 17), generator=g), 7)
    _check_plan(torch.randint(0, 50, (3, 5), generator=g), 60)  # empty buckets
    plan = _check_plan(torch.zeros((60, 60), dtype=torch.int32), 2)  # one long bucket, one empty
    assert plan.multi.tolist() == [[0, 0, -(-3600 // (training._ITEM // 2))]]
    _check_plan(torch.zeros((0, 3), dtype=torch.long), 2)
    index = torch.arange(12).view(3, 4)
    plan = _check_plan(index[:, :2], 12)  # a slice, as of a clamped window
    assert plan.index.is_contiguous() and torch.equal(plan.pairs, index[:, :2].int())


def test_bucket_plan_refusals():
    ok = torch.zeros((2, 2), dtype=torch.long)
    for bad in (ok.float(), ok.bool(), ok[0], ok - 1, ok + 3):
        with pytest.raises(ValueError):
            crumpet.relative_position_buckets(bad, 3)
    with pytest.raises(ValueError):
        crumpet.relative_position_buckets(ok, 0)


def test_cpu_tensors_are_refused():
    plan = crumpet.relative_position_buckets(torch.zeros((8, 8), dtype=torch.long), 1)
    x = torch.zeros(2, 16)
    for call in (lambda: crumpet.relative_position_bias(torch.zeros(1, 2), plan),
                 lambda: crumpet.relative_position_bias_backward(torch.zeros(2, 8, 8), plan),
                 lambda: crumpet.swin_window_attention_train(torch.zeros(1, 8, 3, 2, 16),
                                                             torch.zeros(1, 2), plan),
                 lambda: crumpet.norm_gate_residual(x, x),
                 lambda: crumpet.gelu_checkpoint(x),
                 lambda: crumpet.checkpointed_mlp(x, torch.zeros(4, 16), None, torch.zeros(16, 4),
                                                  None)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_meta_shapes():
    plan = crumpet.relative_position_buckets(torch.zeros((8, 9), dtype=torch.long), 1)
    assert crumpet.relative_position_bias(torch.empty(1, 2, device="meta"), plan).shape == (2, 8, 9)
    x = torch.empty(4, 5, 16, device="meta", dtype=torch.half)
    out, normed = crumpet.norm_gate_residual(x, x.float(), pre_norm=(x[0, 0], x[0, 0]))
    assert out.dtype == torch.float32 and normed.dtype == torch.half and out.shape == x.shape


def test_c_abi_refuses_bad_arguments_without_touching_the_device():
    lib = _ops.capi()
    null, f = ctypes.c_void_p(0), ctypes.c_void_p(16)

    def rejects(rc, code, text):
        assert rc == code and text in _ops.last_error(), (rc, _ops.last_error())

    rejects(lib.crumpet_relative_position_bias(null, 0, null, 0, 5, 2, null, 9, null), 1, "null")
    rejects(lib.crumpet_relative_position_bias(f, 0, f, 7, 5, 2, f, 9, null), 1, "float32")
    rejects(lib.crumpet_relative_position_bias(f, 0, f, 0, 0, 2, f, 9, null), 1, "table_rows")
    assert lib.crumpet_relative_position_bias(null, 0, null, 0, 5, 2, null, 0, null) == 0
    rejects(lib.crumpet_relative_position_bias_backward(f, 0, 2, f, 0, f, 9, null, 3, null, 0,
                                                        null, null), 1, "null")
    rejects(lib.crumpet_relative_position_bias_backward(f, 0, 2, f, 0, f, 9, f, 3, f, 1, null,
                                                        null), 1, "null")

    def backward(shares=1, ws=(7, 7, 7), ss=(0, 0, 0), dtype=2, B=2, H=3, N=343, d=16, scale=0.25,
                 p=f):
        return lib.crumpet_swin_window_attention_qkv_backward(
            p, p, p, p, p, p, 1, 5, p, shares, 1, 1, 1, *ws, *ss, dtype, B, H, N, d, scale, null)

    rejects(backward(p=null), 1, "null")
    rejects(backward(d=48), 3, "head_dim")
    rejects(backward(N=0), 1, "N >= 1")
    rejects(backward(N=50000), 1, "too large")
    rejects(backward(scale=float("nan")), 3, "scale")
    rejects(backward(shares=3), 1, "shares")
    rejects(backward(shares=0), 1, "shares")
    rejects(backward(ss=(7, 0, 0)), 1, "shift")
    rejects(backward(ws=(7, 7, 6), ss=(1, 0, 0)), 1, "geometry")
    rejects(backward(dtype=9), 1, "float32")

    def norm(dtype=2, stream=2, samples=1, M=6, C=16, eps=1e-5, scale=null, post=(null, null)):
        return lib.crumpet_norm_gate_residual(null, null, null, null, dtype, stream, null, scale,
                                              samples, *post, null, null, eps, M, C, null)

    rejects(norm(), 1, "null")
    rejects(norm(stream=1), 1, "stream")
    rejects(norm(C=4097), 1, "4096")
    rejects(norm(eps=0.0), 1, "eps")
    rejects(norm(scale=f, samples=4), 1, "samples")
    rejects(norm(post=(f, null)), 1, "post")
    assert norm(M=0) == 0
    rejects(lib.crumpet_gelu_checkpoint(null, null, null, null, 0, 2, 32, null), 1, "null")
    rejects(lib.crumpet_gelu_checkpoint(null, null, null, null, 0, 2, 1 << 25, null), 1, "2^24")
    assert lib.crumpet_gelu_checkpoint_backward(null, null, null, null, null, 0, 0, 32, null) == 0
    rejects(lib.crumpet_restore_activation(null, null, null, 5, 2, 32, null), 1, "float32")


def test_the_switch_leaves_other_stages_alone():
    """On a model without CUDA the stages keep their own forward, and results."""
    model = swin_unetr.SwinTransformer(1, 16, (4, 4, 4), (2, 2, 2), (1, 1), (1, 2)).train()
    x = torch.randn(1, 1, 16, 16, 16)
    want = model(x)
    assert crumpet.enable_training_kernels(model) == 2
    assert crumpet.enable_training_kernels(model) == 2  # idempotent
    assert all(torch.equal(a, b) for a, b in zip(model(x), want))
    assert crumpet.disable_training_kernels(model) == 2
    assert crumpet.disable_training_kernels(model) == 0
    assert all("forward" not in m.__dict__ for m in model.modules())


def test_which_blocks_train():
    ok = swin_unetr.SwinTransformerBlock(48, 3, (7, 7, 7), (0, 0, 0))
    assert training._block_trains(ok, 48)
    for change in (lambda b: setattr(b.mlp, "fn", torch.nn.GELU("tanh")),
                   lambda b: setattr(b, "use_checkpoint", True),
                   lambda b: setattr(b.attn, "attn_drop", torch.nn.Dropout(0.1)),
                   lambda b: setattr(b, "norm2", torch.nn.LayerNorm(48, elementwise_affine=False)),
                   lambda b: setattr(b, "norm1", torch.nn.BatchNorm1d(48))):
        block = swin_unetr.SwinTransformerBlock(48, 3, (7, 7, 7), (0, 0, 0))
        change(block)
        assert not training._block_trains(block, 48)
    assert not training._block_trains(swin_unetr.SwinTransformerBlock(24, 3, (7, 7, 7), (0, 0, 0)), 24)
