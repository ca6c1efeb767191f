"""The native host path of the feed-forward half's operators beside the Python route: what it serves, what it leaves to the other, and what a caller does around
the operators (checkpoints, compiled callers, autocast, transforms)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("gated_mlp", "gated_mlp_odd", "layer_norm", "residual_layer_norm", "dropout")
NATIVE = {"gated_mlp": "gated_mlp", "gated_mlp_odd": "gated_mlp", "layer_norm": "layer_norm", "residual_layer_norm": "layer_norm", "dropout": "dropout"}


def _calls(dev, dt=BF):
    """name -> (call of a list of tensors, the tensors)."""
    from palimpsa_amd.ops.gated_mlp import gated_mlp
    from palimpsa_amd.ops.layer_glue import dropout, layer_norm, residual_layer_norm
    gen = torch.Generator().manual_seed(3)
    r = lambda *s, t=dt: torch.randn(*s, generator=gen).to(t).to(dev)  # noqa: E731
    B, T, D, F = 2, 37, 64, 96
    norm, seed = [r(B, T, D), r(D, t=F32), r(D, t=F32)], torch.tensor(5, device=dev)
    return {
        "gated_mlp": (lambda a: [gated_mlp(*a)], [r(B, T, D), r(F, D), r(F, D), r(D, F)]),
        "gated_mlp_odd": (lambda a: [gated_mlp(*a, "gelu")], [r(B, T, 61), r(97, 61), r(97, 61), r(39, 97)]),
        "layer_norm": (lambda a: [layer_norm(*a)], norm),
        "residual_layer_norm": (lambda a: list(residual_layer_norm(a[0], a[3], a[1], a[2], dropout_p=0.25, seed=seed, site=3)), norm + [r(B, T, D)]),
        "dropout": (lambda a: [dropout(a[0], 0.25, seed, 3)], [r(B, T, D)]),
    }


def _spied(monkeypatch, native=True):
    from palimpsa_amd import _lib as L
    host, served = L.host(), {}
    for name in set(NATIVE.values()):
        real = getattr(host, name)

        def call(*args, _r=real, _n=name):
            out = _r(*args) if native else None
            served.setdefault(_n, []).append(out is not None)
            return out

        monkeypatch.setattr(host, name, call)
    return served


def _run(call, args, grad=True):
    lv = [t.clone().requires_grad_(grad) for t in args]
    with torch.set_grad_enabled(grad):
        out = list(call(lv))
    if not grad:
        return out
    sum(o.float().square().sum() for o in out).backward()
    return out + [t.grad for t in lv]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("name", NAMES)
def test_routes_agree(gpu_device, monkeypatch, name, dt):
    call, args = _calls(gpu_device, dt)[name]
    for grad in (False, True):
        got = []
        for native in (True, False):
            with monkeypatch.context() as m:
                served = _spied(m, native)
                got.append(_run(call, args, grad))
                assert served == {NATIVE[name]: [native]}
        for x, y in zip(*got):
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(gpu_device, monkeypatch, name, native):
    import torch.autograd.forward_ad as fw
    _spied(monkeypatch, native)
    call, args = _calls(gpu_device)[name]
    for which in range(len(args)):
        for grad in (False, True):
            with fw.dual_level(), torch.set_grad_enabled(grad):
                a = [t.clone() for t in args]
                a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
                with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
                    call(a)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_gradients_are_not_differentiated_again(gpu_device, monkeypatch, name, native):
    _spied(monkeypatch, native)
    call, args = _calls(gpu_device, F32)[name]
    lv = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(call(lv)[0].square().sum(), lv[:2], create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError):
            g.sum().backward(retain_graph=True)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_activation_checkpointing(gpu_device, monkeypatch, name, reentrant, native):
    from torch.utils.checkpoint import checkpoint
    _spied(monkeypatch, native)
    call, args = _calls(gpu_device)[name]
    want = _run(call, args)
    got = _run(lambda a: checkpoint(lambda *t: tuple(call(list(t))), *a, use_reentrant=reentrant), args)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_modes_and_transforms_take_the_python_route(gpu_device, monkeypatch):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    served = _spied(monkeypatch)
    for name, (call, args) in _calls(gpu_device).items():
        with torch.no_grad():
            want = call(args)
            assert served.pop(NATIVE[name]) == [True]
            with Mode():
                got = call(args)
        assert served.pop(NATIVE[name]) == [False] and all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(RuntimeError):                     # no rule for a batch of calls: an error, not a result without one
            torch.func.vmap(lambda t: call([t] + args[1:])[0])(args[0][None])
        assert not any(served.pop(NATIVE[name], []))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call([t] + args[1:])[0].float().sum())(args[0])
        assert not any(served.pop(NATIVE[name], []))


@pytest.mark.parametrize("name", NAMES)
def test_compiled_caller(gpu_device, name):
    call, args = _calls(gpu_device)[name]
    torch._dynamo.reset()
    compiled = torch.compile(lambda a: call(a), backend="eager")
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(compiled(args), call(args)))
    torch._dynamo.reset()
    assert all(torch.equal(x, y) for x, y in zip(_run(torch.compile(lambda a: call(a), backend="eager"), args), _run(call, args)))


@pytest.mark.parametrize("name", NAMES)
def test_autocast_changes_nothing(gpu_device, name):
    """The operators take the types that they are given: rows in bf16 with weights in fp32 are computed from fp32 under autocast too."""
    call, args = _calls(gpu_device)[name]
    for a in (args, [args[0]] + [t.float() for t in args[1:]], [t.float() for t in args]):
        want = _run(call, a)
        with torch.autocast("cuda", dtype=BF):
            lv = [t.clone().requires_grad_(True) for t in a]
            out = call(lv)
        got = out + list(torch.autograd.grad(sum(o.float().square().sum() for o in out), lv))
        for x, y, t in zip(got, want, [None] * len(out) + a):
            assert x.dtype == y.dtype and torch.equal(x, y) and (t is None or x.dtype == t.dtype)


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(gpu_device, name):
    call, args = _calls(gpu_device)[name]
    want = _run(call, args, False)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(call([t.clone() for t in args]), want))


@pytest.mark.parametrize("name", NAMES)
def test_a_graph_that_is_walked_twice(gpu_device, name):
    call, args = _calls(gpu_device)[name]
    lv = [t.clone().requires_grad_(True) for t in args]
    out = call(lv)
    loss = sum(o.float().square().sum() for o in out)
    first, second = torch.autograd.grad(loss, lv, retain_graph=True), torch.autograd.grad(loss, lv)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
