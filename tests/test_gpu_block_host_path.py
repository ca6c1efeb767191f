"""The native host path of the residual norm, the short convolution and the selective scan against the Python route: the same kernels on
the same values, so results, states and gradients are equal bit for bit; what the native path has no business with goes to the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls(dev, dt=torch.bfloat16, packed=False, wdt=torch.float32):
    """name of the native function -> (call of the public entry point on a dict of tensors, its tensors, whether it has gradients)."""
    from palimpsa_amd.ops.layer_glue import residual_rms_norm, residual_rms_norm_fp8
    from palimpsa_amd.ops.selective_scan import selective_scan, selective_scan_step
    from palimpsa_amd.ops.short_conv import short_conv, short_conv_step
    gen = torch.Generator().manual_seed(3)
    r = lambda *s, t=dt: torch.randn(*s, generator=gen).to(t).to(dev)  # noqa: E731
    B, T, D, W, N, G = (1, 90, 40, 4, 16, 2) if packed else (2, 37, 40, 4, 16, 2)
    cu = torch.tensor([0, 0, 33, 34, 90], device=dev) if packed else None
    S = 4 if packed else B
    norm = dict(x=r(B, T, 128), residual=r(B, T, 128), weight=r(128, t=wdt))
    conv = dict(x=r(B, T, D), weight=r(D, W, t=wdt) / 2, bias=r(D, t=wdt), initial_state=r(S, D, W))
    rows = dict(u=r(B, T, D), delta=r(B, T, D), B=r(B, T, G, N), C=r(B, T, G, N), z=r(B, T, D))
    par = dict(A=-torch.rand(D, N, generator=gen).to(dev) - .1, D=r(D, t=torch.float32), delta_bias=r(D, t=torch.float32))
    one = {n: t[:, 0].contiguous() for n, t in rows.items()}
    f32 = torch.float32
    return {
        "residual_norm": (lambda a: residual_rms_norm(**a), norm, True),
        "residual_norm_fp8": (lambda a: residual_rms_norm_fp8(**a, group_size=64), norm, False),
        "short_conv": (lambda a: short_conv(**a, output_final_state=True, cu_seqlens=cu), conv, True),
        "short_conv_step": (lambda a: (short_conv_step(**a), a["state"]),
                            dict(x=r(B, D), state=r(B, D, W), weight=conv["weight"], bias=conv["bias"]), False),
        "selective_scan": (lambda a: selective_scan(**a, output_final_state=True, cu_seqlens=cu),
                           dict(rows, **par, initial_state=r(S, D, N, t=f32)), True),
        "selective_scan_step": (lambda a: (selective_scan_step(**a), a["state"]), dict(one, **par, state=r(B, D, N, t=f32)), False),
    }


def _spied(monkeypatch, native=True):
    from palimpsa_amd import _lib as L
    host, served = L.host(), {}
    for name in _NAMES:
        real = getattr(host, name)

        def call(*args, _r=real, _n=name):
            out = _r(*args) if native else None
            served.setdefault(_n, []).append(out is not None)
            return out

        monkeypatch.setattr(host, name, call)
    return served


_NAMES = ("residual_norm", "residual_norm_fp8", "short_conv", "short_conv_step", "selective_scan", "selective_scan_step")


def _run(call, args, grad, without=()):
    lv = {n: t.clone().requires_grad_(grad and n not in without) for n, t in args.items()}
    with torch.set_grad_enabled(grad):
        out = list(call(lv))
    if grad:
        out += torch.autograd.grad(sum(o.float().square().sum() for o in out), [t for t in lv.values() if t.requires_grad])
    return out


@pytest.mark.parametrize("dt,wdt,packed", [(torch.bfloat16, torch.float32, False), (torch.float32, torch.float32, True),
                                           (torch.bfloat16, torch.bfloat16, True)])
@pytest.mark.parametrize("name", _NAMES)
def test_routes_agree(gpu_device, monkeypatch, name, dt, wdt, packed):
    call, args, has_grad = _calls(gpu_device, dt, packed, wdt)[name]
    for grad in (False, True)[:1 + has_grad]:
        for without in ((), ("initial_state", "residual")):
            with monkeypatch.context() as m:
                served = _spied(m)
                a = _run(call, args, grad, without)
                assert served == {name: [True]}
            with monkeypatch.context() as m:
                served = _spied(m, native=False)
                b = _run(call, args, grad, without)
                assert served == {name: [False]}
            assert len(a) == len(b)
            for x, y in zip(a, b):
                assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_strided_rows_are_read_where_they_are(gpu_device, monkeypatch):
    served = _spied(monkeypatch)
    for name in ("residual_norm", "short_conv", "selective_scan"):
        call, args, _ = _calls(gpu_device)[name]
        rows = ("x",) if name != "selective_scan" else ("u", "delta", "B", "z")
        wide = {n: (torch.cat([t, t, t], -1)[..., :t.shape[-1]] if n in rows and n != "B" else t) for n, t in args.items()}
        for a, b in zip(_run(call, args, True), _run(call, wide, True)):
            assert torch.equal(a, b)
    assert all(all(s) for s in served.values()) and len(served) == 3


@pytest.mark.parametrize("name", _NAMES)
def test_forward_mode_is_refused(gpu_device, name):
    import torch.autograd.forward_ad as fw
    call, args, _ = _calls(gpu_device)[name]
    for grad in (False, True):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            a = {n: t.clone() for n, t in args.items()}
            n = next(iter(a))
            a[n] = fw.make_dual(a[n], torch.ones_like(a[n]))
            with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
                call(a)


@pytest.mark.parametrize("name", [n for n in _NAMES if "step" in n or "fp8" in n])
def test_calls_without_gradients_refuse_them(gpu_device, name):
    call, args, _ = _calls(gpu_device)[name]
    a = {n: t.clone() for n, t in args.items()}
    a["weight" if "weight" in a else "A"].requires_grad_(True)
    with pytest.raises((ValueError, RuntimeError)):
        call(a)
    with torch.no_grad():
        call(a)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["residual_norm", "short_conv", "selective_scan"])
def test_gradients_are_not_differentiated_again(gpu_device, monkeypatch, name, native):
    _spied(monkeypatch, native)
    call, args, _ = _calls(gpu_device, torch.float32)[name]
    lv = {n: t.clone().requires_grad_(True) for n, t in args.items()}
    first = next(iter(lv.values()))
    g, = torch.autograd.grad(call(lv)[0].square().sum(), first, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("name", ["residual_norm", "short_conv", "selective_scan"])
def test_saved_tensors_go_through_hooks(gpu_device, name):
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    call, args, _ = _calls(gpu_device)[name]
    want = _run(call, args, True)
    with save_on_cpu():
        got = _run(call, args, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for change in (lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu()):
        lv = {n: t.clone().requires_grad_(True) for n, t in args.items()}
        with saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dim() > 2 and t.dtype == torch.bfloat16 else t):
            out = call(lv)
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad(out[0].float().sum(), list(lv.values()))


@pytest.mark.parametrize("name", ["residual_norm", "short_conv", "selective_scan"])
def test_activation_checkpointing(gpu_device, name):
    from torch.utils.checkpoint import checkpoint
    call, args, _ = _calls(gpu_device)[name]
    want = _run(call, args, True)
    names = list(args)
    got = _run(lambda a: checkpoint(lambda *t: tuple(call(dict(zip(names, t)))), *a.values(), use_reentrant=False), args, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_states_written_in_place_count_as_written(gpu_device):
    for name in ("short_conv_step", "selective_scan_step"):
        call, args, _ = _calls(gpu_device)[name]
        v = args["state"]._version
        call(args)
        assert args["state"]._version > v
        w = torch.ones_like(args["state"]).requires_grad_(True)
        kept = (w * args["state"]).sum()
        call(args)
        with pytest.raises(RuntimeError):
            kept.backward()
        with torch.inference_mode():
            call({n: t.clone() for n, t in args.items()})


def test_modes_and_transforms_take_the_python_route(gpu_device, monkeypatch):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    served = _spied(monkeypatch)
    for name, (call, args, _) in _calls(gpu_device).items():
        with Mode(), torch.no_grad():
            call(args)
        assert served.pop(name) == [False]


def test_compiled_caller(gpu_device):
    """A caller under torch.compile breaks its graph at the operators and gets what the eager caller gets."""
    for name in ("residual_norm", "short_conv", "selective_scan"):
        call, args, _ = _calls(gpu_device)[name]
        torch._dynamo.reset()
        compiled = torch.compile(lambda a, c=call: c(a), backend="eager")
        with torch.no_grad():
            assert all(torch.equal(x, y) for x, y in zip(compiled(args), call(args)))
