"""Saved tensors of the feed-forward half's operators that go through hooks, on both routes: what comes back with other strides is read where it
lies, what comes back in another size, type or place is refused before anything is launched."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _calls(dev, dt=BF):
    """name -> (call of a list of leaves on the native route, on the Python route, the leaves); x and residual are slices of wider rows."""
    from palimpsa_amd.ops import layer_glue as lg
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    gen = torch.Generator().manual_seed(11)
    r = lambda *s, t=dt: torch.randn(*s, generator=gen).to(t).to(dev)  # noqa: E731
    B, T, D, F, Do = 2, 37, 64, 96, 40
    wide = lambda: r(B, T, 3 * D)[..., D:2 * D]  # noqa: E731
    seed = torch.tensor(77, device=dev)
    norm = [wide(), r(D, t=F32), r(D, t=F32)]
    return {
        "gated_mlp": (lambda a: [gated_mlp(*a)], lambda a: [_gated_mlp(*a, "silu")], [wide(), r(F, D), r(F, D), r(Do, F)]),
        "gated_mlp_odd": (lambda a: [gated_mlp(*a)], lambda a: [_gated_mlp(*a, "silu")], [wide()[..., :61], r(97, 61), r(97, 61), r(39, 97)]),
        "layer_norm": (lambda a: [lg.layer_norm(*a)], lambda a: [lg._layer_norm(a[0], None, a[1], a[2], 1e-5, False, False, 0.0, 0, None, 0)], norm),
        "residual_layer_norm": (lambda a: list(lg.residual_layer_norm(a[0], a[3], a[1], a[2], dropout_p=0.25, seed=seed, site=3)),
                                lambda a: list(lg._layer_norm(a[0], a[3], a[1], a[2], 1e-5, False, True, 0.25, 0, seed, 3)), norm + [wide()]),
        "dropout": (lambda a: [lg.dropout(a[0], 0.25, seed, 3)], lambda a: [lg._dropout(a[0], 0.25, seed, 3)], [wide()]),
    }


NAMES = ("gated_mlp", "gated_mlp_odd", "layer_norm", "residual_layer_norm", "dropout")


def _leaves(args):
    return [t.detach().requires_grad_(True) for t in args]        # (a slice stays one)


def _grads(out, leaves):
    return [o.detach() for o in out] + list(torch.autograd.grad(sum(o.float().square().sum() for o in out), leaves))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_tensors_that_were_on_the_host_in_between(gpu_device, name, native):
    both = _calls(gpu_device)[name]
    call, args = both[0 if native else 1], both[2]
    leaves = _leaves(args)
    assert name == "dropout" or not leaves[0].is_contiguous()
    want = _grads(call(leaves), leaves)
    with save_on_cpu():
        out = call(leaves)
    for a, b in zip(_grads(out, leaves), want):
        assert torch.equal(a, b)


def _twice(t):
    return torch.cat([t, t]) if t.dim() else torch.stack([t, t])


CHANGES = {"twice": _twice, "a part": lambda t: t[:1] if t.dim() and t.shape[0] > 1 else t[None].expand(2), "double": lambda t: t.double(), "on the host": lambda t: t.cpu()}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_a_saved_tensor_that_came_back_otherwise_is_refused(gpu_device, name, native):
    both = _calls(gpu_device)[name]
    call, args = both[0 if native else 1], both[2]
    saved = []
    with saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        call(_leaves(args))
    for which in range(len(saved)):
        for how, change in CHANGES.items():
            print(name, native, which, how, flush=True)
            leaves, n = _leaves(args), []
            with saved_tensors_hooks(lambda t: n.append(0) or (len(n) - 1, t), lambda p: change(p[1]) if p[0] == which else p[1]):
                out = call(leaves)
            with pytest.raises((ValueError, RuntimeError), match="came back|same device|must be on"):
                torch.autograd.grad(out[0].float().sum(), leaves)


@pytest.mark.parametrize("native", [True, False])
def test_changes_that_agree_with_each_other_are_refused_too(gpu_device, native):
    """Rows and parameters as long as each other, but not as long as the gradient that comes in."""
    wider = lambda t: torch.cat([t, t], -1) if t.dtype != F32 or t.dim() == 1 else t  # noqa: E731
    higher = lambda t: torch.cat([t, t]) if t.dim() > 1 else t  # noqa: E731
    for name, change in (("layer_norm", wider), ("layer_norm", higher), ("residual_layer_norm", wider), ("residual_layer_norm", higher)):
        both = _calls(gpu_device)[name]
        leaves = _leaves(both[2])
        with saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype != torch.int64 else t):
            out = both[0 if native else 1](leaves)
        with pytest.raises(ValueError, match="came back"):
            torch.autograd.grad(out[0].float().sum(), leaves)


@pytest.mark.parametrize("native", [True, False])
def test_few_rows_whose_kept_numbers_fill_no_more_room(gpu_device, native):
    """Three rows of eight hidden entries and six of them are kept in the same 256 bytes: the sizes of the gradient tell them apart."""
    from palimpsa_amd.ops.gated_mlp import _gated_mlp, gated_mlp
    gen = torch.Generator().manual_seed(1)
    leaves = [torch.randn(*s, generator=gen).to(BF).to(gpu_device).requires_grad_(True) for s in ((3, 8), (8, 8), (8, 8), (8, 8))]
    for at in (0, 3):
        n = []
        with saved_tensors_hooks(lambda t: n.append(0) or (len(n) - 1, t), lambda p: torch.cat([p[1], p[1]]) if p[0] == at else p[1]):
            y = gated_mlp(*leaves) if native else _gated_mlp(*leaves, "silu")
        with pytest.raises(ValueError, match="came back"):
            torch.autograd.grad(y.float().sum(), leaves)
