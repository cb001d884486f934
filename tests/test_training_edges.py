"""Training operators, what needs no GPU: which blocks the switch takes, how a switched model
copies, and what the functions refuse."""

from __future__ import annotations

import pytest
import torch

import crumpet_b200 as crumpet
from crumpet_b200 import swin_unetr, training


def block():
    return swin_unetr.SwinTransformerBlock(48, 3, (7, 7, 7), (0, 0, 0)).train()


class Adapter(torch.nn.Linear):
    """A Linear with a low-rank addition."""

    def __init__(self, *a):
        super().__init__(*a)
        self.down = torch.nn.Parameter(torch.randn(2, self.in_features))
        self.up = torch.nn.Parameter(torch.randn(self.out_features, 2))

    def forward(self, x):
        return super().forward(x) + x @ self.down.t() @ self.up.t()


class Wrapped(torch.nn.Module):
    """A Linear held by another module that shows its parameters."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    weight = property(lambda self: self.inner.weight)
    bias = property(lambda self: self.inner.bias)

    def forward(self, x):
        return 2 * self.inner(x)


class Norm(torch.nn.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 1


class Double(torch.nn.Module):
    def forward(self, weight):
        return 2 * weight


class Block(swin_unetr.SwinTransformerBlock):
    def forward(self, x, mask_matrix):
        return 2 * super().forward(x, mask_matrix)


class Mlp(swin_unetr.MLPBlock):
    def forward(self, x):
        return 2 * super().forward(x)


def prune(linear):
    import torch.nn.utils.prune as prune

    prune.l1_unstructured(linear, "weight", 0.5)


CHANGES = {
    "adapter": lambda b: setattr(b.mlp, "linear1", Adapter(48, 192)),
    "wrapped": lambda b: setattr(b.mlp, "linear2", Wrapped(b.mlp.linear2)),
    "weight norm": lambda b: torch.nn.utils.weight_norm(b.mlp.linear1),
    "parametrized": lambda b: torch.nn.utils.parametrize.register_parametrization(
        b.mlp.linear1, "weight", Double()),
    "pruned": lambda b: prune(b.mlp.linear2),
    "norm subclass": lambda b: setattr(b, "norm2", Norm(48)),
    "first norm": lambda b: setattr(b, "norm1", Norm(48)),
    "block subclass": lambda b: setattr(b, "__class__", Block),
    "mlp subclass": lambda b: setattr(b.mlp, "__class__", Mlp),
    "own forward": lambda b: setattr(b.mlp, "forward", lambda x: x),
    "other softmax": lambda b: setattr(b.attn, "softmax", torch.nn.Softmax(-2)),
    "hook": lambda b: b.mlp.linear2.register_forward_hook(lambda *a: None),
    "pre-hook": lambda b: b.norm2.register_forward_pre_hook(lambda *a: None),
    "hook on the block": lambda b: b.register_forward_hook(lambda *a: None),
    "hook on the attention": lambda b: b.attn.register_forward_hook(lambda *a: None),
    "gradient hook": lambda b: b.mlp.register_full_backward_hook(lambda *a: None),
    "gradient pre-hook": lambda b: b.mlp.fn.register_full_backward_pre_hook(lambda *a: None),
    "drop path subclass": lambda b: setattr(b, "drop_path", MyDropPath()),
}


class DropPath(torch.nn.Module):
    drop_prob, scale_by_keep = 0.5, True


class MyDropPath(DropPath):
    def forward(self, x):
        return -x


@pytest.mark.parametrize("what", CHANGES)
def test_blocks_of_other_modules_keep_their_forward(what):
    """The kernels read these modules' parameters without calling them."""
    b = block()
    assert training._block_trains(b, 48)
    CHANGES[what](b)
    assert not training._block_trains(b, 48)


def test_modules_that_are_called_may_be_any():
    """qkv and proj are called as modules, their hooks run."""
    b = block()
    b.attn.qkv = Adapter(48, 144)
    b.attn.proj.register_forward_hook(lambda *a: None)
    b.drop_path = DropPath()
    assert training._block_trains(b, 48)


def test_global_hooks():
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        assert not training._block_trains(block(), 48)
    finally:
        handle.remove()
    assert training._block_trains(block(), 48)


def test_drop_path_of_a_block_in_eval_mode():
    b = block()
    b.drop_path = DropPath()
    assert training._path_scale(b, 4, "cpu") is not None
    b.eval()
    assert training._path_scale(b, 4, "cpu") is None


def stage():
    return swin_unetr.BasicLayer(48, 2, 3, (4, 4, 4)).train()


def copies(layer):
    """Replicas, deep copies and pickles of a stage."""
    import copy
    import io
    import pickle

    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    return {"replica": layer._replicate_for_data_parallel(), "deepcopy": copy.deepcopy(layer),
            "copy": copy.copy(layer), "pickle": pickle.loads(pickle.dumps(layer)),
            "file": torch.load(file, weights_only=False)}


def test_copies_of_a_switched_stage_are_their_own(monkeypatch):
    layer = stage()
    x = torch.randn(1, 48, 4, 8, 4)
    want = layer(x)
    assert crumpet.enable_training_kernels(layer) == 1
    for name, other in copies(layer).items():
        assert other is not layer and isinstance(other, swin_unetr.BasicLayer), name
        assert torch.equal(other(x), want), name  # on the CPU: the copy's own forward
        assert type(other) is type(layer), name
    monkeypatch.setattr(training, "_stage_trains", lambda layer, x: True)
    monkeypatch.setattr(training, "_train_layer", lambda layer, x, size: layer)
    for name, other in copies(layer).items():
        assert other(x) is other, name
        assert crumpet.disable_training_kernels(other) == 1, name
        assert type(other) is swin_unetr.BasicLayer and torch.equal(other(x), want), name
    assert layer(x) is layer
    assert repr(layer).startswith("BasicLayer(")


def test_a_stage_switched_back_leaves_no_trace():
    import pickle

    layer = stage()
    before = pickle.dumps(layer)
    crumpet.enable_training_kernels(layer)
    training._module_buckets(layer.blocks[0].attn, 64)
    assert training._module_buckets(layer.blocks[0].attn, 64) \
        is training._module_buckets(layer.blocks[0].attn, 64)
    crumpet.disable_training_kernels(layer)
    assert pickle.dumps(layer) == before


def test_the_patch_and_the_switch_in_either_order():
    x = torch.randn(1, 48, 8, 8, 8)
    layer, other = stage(), stage()
    other.load_state_dict(layer.state_dict())
    want = layer(x)
    crumpet.enable_training_kernels(layer)
    assert crumpet.patch_monai_swin_unetr(swin_unetr)
    try:
        crumpet.enable_training_kernels(other)
        for m in (layer, other):
            assert type(m)._crumpet_stage.forward is swin_unetr.BasicLayer.forward
    finally:
        crumpet.unpatch_monai_swin_unetr()
    assert torch.equal(layer(x), want) and torch.equal(other(x), want)


def test_a_stage_with_its_own_forward_is_left_alone():
    layer = stage()
    layer.forward = lambda x: x + 1
    assert crumpet.enable_training_kernels(layer) == 0
    x = torch.zeros(1)
    assert torch.equal(layer(x), x + 1)


def test_buckets_follow_the_index():
    """Laid out again for an index that was written to or replaced, and not kept with the module."""
    attn = block().attn
    first = training._module_buckets(attn, 343)
    assert training._module_buckets(attn, 343) is first
    attn.relative_position_index[0, 0] = 0
    again = training._module_buckets(attn, 343)
    assert again is not first and int(again.pairs[0, 0]) == 0
    attn.relative_position_index = attn.relative_position_index.clone()
    assert training._module_buckets(attn, 343) is not again


def dual_calls(device):
    """Every operator on a tensor with a tangent that needs no gradient, and none recorded."""
    from crumpet_b200 import _ops

    ops = _ops.require()
    plan = crumpet.relative_position_buckets(torch.zeros((8, 8), dtype=torch.long, device=device), 1)
    d = lambda *s: torch.autograd.forward_ad.make_dual(  # noqa: E731
        torch.ones(s, device=device), torch.ones(s, device=device))
    x, qkv, table = d(4, 32), d(1, 8, 3, 2, 16), d(1, 2)
    kept = torch.ones((4, 32), dtype=torch.int8, device=device)
    scales = torch.ones((4, 1), dtype=torch.uint8, device=device)
    place = [1, 1, 1], [2, 2, 2], [0, 0, 0], 0.25
    yield lambda: ops.relative_position_bias(table, plan.pairs, torch.float32)
    yield lambda: ops.relative_position_bias_backward(d(2, 8, 8), *plan[2:5], 1, torch.float32)
    yield lambda: ops.swin_window_attention_train(qkv, table, *plan[:2], *place)
    yield lambda: ops.swin_window_attention_train(qkv.detach(), table, *plan[:2], *place)
    yield lambda: ops.swin_window_attention_backward(d(1, 8, 32), qkv, table, *plan[1:5], *place)
    yield lambda: ops.norm_gate_residual(x, x, None, None, None, None, None, None, 1e-5)
    yield lambda: ops.norm_gate_residual(torch.ones_like(x).detach(), torch.ones_like(x).detach(),
                                         d(32), None, None, None, None, None, 1e-5)
    yield lambda: ops.norm_gate_residual_backward(x, None, x, x, None, None, None, None, None, 1e-5)
    yield lambda: ops.gelu_checkpoint(x)
    yield lambda: ops.gelu_checkpoint_backward(x, kept, scales)


def test_tangents_are_refused():
    """A result without its tangent would be a derivative of zero."""
    with torch.autograd.forward_ad.dual_level():
        for i, call in enumerate(dual_calls("cpu")):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        from crumpet_b200 import _ops

        torch.func.jvp(lambda x: _ops.require().gelu_checkpoint(x)[0], (torch.ones(2, 32),),
                       (torch.ones(2, 32),))


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_a_plan_does_not_change_with_the_index(dtype):
    index = torch.arange(12, dtype=dtype).view(3, 4)
    plan = crumpet.relative_position_buckets(index, 12)
    index.fill_(99)
    assert torch.equal(plan.index, torch.arange(12).view(3, 4))
    assert torch.equal(plan.pairs, plan.index.int())


def plain_gelu(monkeypatch):
    """The 8-bit GELU's calls in plain torch, for what is around them."""
    def keep(x):
        return torch.nn.functional.gelu(x), training.KeptActivation(x, x, x.dtype)

    def back(grad, kept):
        u = kept.kept.detach().requires_grad_(True)
        with torch.enable_grad():
            y = torch.nn.functional.gelu(u)
        return torch.autograd.grad(y, u, grad)[0], y.detach()

    monkeypatch.setattr(training, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(training, "gelu_checkpoint", keep)
    monkeypatch.setattr(training, "gelu_checkpoint_backward", back)


@pytest.mark.parametrize("frozen", [(), (1, 2, 3, 4), (1, 2), (3, 4), (0,), (0, 1, 2), (0, 1, 3), (0, 2, 4),
                                    (0, 1, 2, 3)], ids=str)
def test_mlp_takes_the_products_that_are_asked_for(monkeypatch, frozen):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        products = sums = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.products += func.overloadpacket in (torch.ops.aten.mm, torch.ops.aten.addmm)
            self.sums += func.overloadpacket == torch.ops.aten.sum
            return func(*args, **(kwargs or {}))

    plain_gelu(monkeypatch)
    g = torch.Generator().manual_seed(0)
    args = [torch.randn(s, generator=g) for s in ((5, 16), (64, 16), (64,), (16, 64), (16,))]
    for i, t in enumerate(args):
        t.requires_grad_(i not in frozen)
    x, w1, b1, w2, b2 = args
    want = torch.nn.functional.linear(torch.nn.functional.gelu(
        torch.nn.functional.linear(x, w1, b1)), w2, b2)
    got = crumpet.checkpointed_mlp(*args)
    torch.testing.assert_close(got, want)
    asked = [t for t in args if t.requires_grad]
    grad = torch.randn(want.shape, generator=g)
    wanted = torch.autograd.grad(want, asked, grad)
    with Count() as count:
        grads = torch.autograd.grad(got, asked, grad)
    for a, b in zip(grads, wanted):
        torch.testing.assert_close(a, b)
    on = [t.requires_grad for t in args]
    assert count.products == any(on[:4]) + on[0] + on[1] + on[3]
    assert count.sums == on[2] + on[4]


def test_eight_bit_activations_are_a_choice(monkeypatch):
    kept = []
    monkeypatch.setattr(training, "checkpointed_mlp", lambda x, *a: kept.append(1) or x)
    monkeypatch.setattr(training, "_stage_trains", lambda layer, x: True)
    monkeypatch.setattr(training, "_train_branch", lambda blk, normed, *a: normed)
    monkeypatch.setattr(training, "norm_gate_residual",
                        lambda b, x, **k: (b + x, b if k["pre_norm"] else None))
    layer = stage()
    called = []
    x = torch.randn(1, 48, 4, 4, 4)
    for on in (True, False, True):
        crumpet.enable_training_kernels(layer, on)
        kept.clear(), called.clear()
        handles = [b.mlp.register_forward_hook(lambda *a: called.append(1)) for b in layer.blocks]
        layer(x)
        assert (len(kept), len(called)) == ((2, 0) if on else (0, 2))
        for h in handles:
            h.remove()
    for other in copies(crumpet.enable_training_kernels(layer, False) and layer).values():
        kept.clear()
        other(x)
        assert not kept
