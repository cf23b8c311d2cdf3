"""The low-bit operators on the CPU: schemas, shapes, refusals, argument checks of the C ABI (nothing here launches a kernel)."""
import ctypes

import pytest
import torch

from prime_amd import lowbit
from tests import lowbit_reference as ref


def test_every_lowbit_op_traces_on_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, r, w = torch.empty(2, 3, 70, dtype=torch.bfloat16), torch.empty(2, 3, 70, dtype=torch.bfloat16), torch.empty(70)
        codes, scales, inv = lowbit.rms_norm_quantize(x, w)
        assert codes.shape == (2, 3, 70) and codes.dtype == torch.int8 and scales.shape == inv.shape == (2, 3)
        codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(x, r, w, 1e-5, torch.float8_e4m3fn)
        assert codes.dtype == torch.float8_e4m3fn and hidden.shape == x.shape and hidden.dtype == torch.bfloat16
        assert scales.dtype == inv.dtype == torch.float32
        gx, gw = lowbit.rms_norm_quantize_backward(x, hidden, w, inv, r)
        assert gx.shape == x.shape and gx.dtype == torch.bfloat16 and gw.shape == (70,) and gw.dtype == torch.float32
        packed, s = lowbit.quantize_4bit(torch.empty(5, 70), 32, torch.float32)
        assert packed.shape == (5, 48) and packed.dtype == torch.uint8 and s.shape == (5, 3) and s.dtype == torch.float32
        assert lowbit.dequantize_4bit(packed, s, 70, torch.float16).shape == (5, 70)
        assert lowbit.dequantize_4bit(packed, s).shape == (5, 96)
        y = lowbit.matvec_4bit(x, packed, s)
        assert y.shape == (2, 3, 5) and y.dtype == torch.bfloat16
        assert lowbit.matvec_4bit(codes.to(torch.int8), packed, s, scales).dtype == torch.float32
    names = {s.name.split("::")[1] for s in torch._C._jit_get_all_schemas() if s.name.startswith("prime_lowbit::")}
    assert names == {"rms_norm_quantize", "add_rms_norm_quantize", "rms_norm_quantize_backward", "quantize_4bit", "dequantize_4bit", "matvec_4bit"}


def test_cpu_tensors_reach_no_kernel():
    x, w = torch.randn(3, 64), torch.ones(64)
    packed, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1)
    for call in (lambda: lowbit.rms_norm_quantize(x, w), lambda: lowbit.add_rms_norm_quantize(x, x, w),
                 lambda: lowbit.rms_norm_quantize_backward(x, x, w, torch.ones(3)), lambda: lowbit.quantize_4bit(x, 64),
                 lambda: lowbit.dequantize_4bit(packed, s), lambda: lowbit.matvec_4bit(x, packed, s)):
        with pytest.raises(NotImplementedError):
            call()


def _refusals():
    """(what is wrong, the implementation behind the dispatcher, arguments): the checks come before anything touches a device."""
    x, w = torch.randn(3, 64), torch.ones(64)
    packed, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1)
    n, a, b = lowbit._rms_norm_quantize, lowbit._add_rms_norm_quantize, lowbit._rms_norm_quantize_backward
    q, d, m = lowbit._quantize_4bit, lowbit._dequantize_4bit, lowbit._matvec_4bit
    i8 = torch.zeros(3, 64, dtype=torch.int8)
    return [
        ("Float, BFloat16 or Half", n, (x.double(), w)), ("1 to 2\\^30", n, (torch.tensor(1.0), w)), ("1 to 2\\^30", n, (x[:, :0], w[:0])),
        ("weight needs shape", n, (x, w[:63])), ("weight needs shape", n, (x, w.view(1, 64))), ("weight must be", n, (x, w.half())),
        ("codes are", n, (x, w, 1e-6, torch.uint8)), ("eps", n, (x, w, -1e-6)), ("eps", n, (x, w, float("nan"))),
        ("residual must have", a, (x, x[:2], w)), ("residual must have", a, (x, x.half(), w)),
        ("no gradient", n, (x, torch.nn.Parameter(w))), ("no gradient", a, (x, x.clone().requires_grad_(), w)),
        ("grad must have", b, (x[:2], x, w, torch.ones(3))), ("inv_rms must be", b, (x, x, w, torch.ones(2))),
        ("inv_rms must be", b, (x, x, w, torch.ones(3).double())), ("grad_hidden must have", b, (x, x, w, torch.ones(3), x.half())),
        ("Float, BFloat16 or Half weight", q, (packed,)), ("a matrix", q, (w,)), ("a matrix", q, (x[:, :0],)), ("group size", q, (x, 48)),
        ("scales are", q, (x, 64, torch.float16)),
        ("Byte codes", d, (packed.int(), s)), ("Byte codes", d, (packed, s.half())), ("same rows", d, (packed, s[:3])), ("same rows", d, (packed, s[:, :0])),
        ("do not make groups", d, (packed, torch.ones(4, 3))), ("do not make groups", d, (packed, torch.ones(4, 4))), ("hold 1 to 64", d, (packed, s, 65)),
        ("hold 1 to 64", d, (packed, s, 0)), ("hold 33 to 64", d, (packed, torch.ones(4, 2), 32)), ("weights are", d, (packed, s, 64, torch.int8)),
        ("Char rows", m, (x.double(), packed, s)), ("a scalar", m, (torch.tensor(1.0), packed, s)), ("hold 1 to 64", m, (torch.randn(3, 65), packed, s)),
        ("come with x_scales", m, (i8, packed, s)), ("come with x_scales", m, (x, packed, s, torch.ones(3))),
        ("x_scales must be", m, (i8, packed, s, torch.ones(2))), ("x_scales must be", m, (i8, packed, s, torch.ones(3).half())),
        ("products are", m, (x, packed, s, None, torch.int8)), ("no gradient", m, (x.clone().requires_grad_(), packed, s)),
    ]


@pytest.mark.parametrize("case", range(len(_refusals())))
def test_refusals(case):
    what, call, args = _refusals()[case]
    with pytest.raises(RuntimeError, match=what):
        call(*args)


def test_tensors_on_two_devices_are_refused():
    x, w = torch.empty(3, 64, device="meta"), torch.ones(64)
    with pytest.raises(RuntimeError, match="one device"):
        lowbit._rms_norm_quantize(x, w)


def test_c_abi_refuses_bad_arguments_before_any_launch():
    from prime_amd import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(4096)

    def norm(x=p, xs=64, r=None, rs=0, w=p, rows=3, dim=64, t=0, wt=0, ct=3, eps=1e-6, codes=p, scales=p, hidden=None, inv=p):
        return lib.prime_rms_norm_quantize(x, xs, r, rs, w, rows, dim, t, wt, ct, eps, codes, scales, hidden, inv, None)

    assert norm(rows=0, x=None) == 0
    for bad in (dict(x=None), dict(w=None), dict(codes=None), dict(scales=None), dict(inv=None), dict(r=p), dict(hidden=p), dict(rows=-1), dict(dim=0),
                dict(dim=(1 << 30) + 1), dict(t=3), dict(wt=1), dict(ct=0), dict(eps=-1.0), dict(eps=float("nan")), dict(xs=-1)):
        assert norm(**bad) == -1, bad
        assert b"prime_rms_norm_quantize" in lib.prime_hip_last_error()
    need = lib.prime_rms_norm_backward_scratch_bytes(3, 64)
    assert need >= 64 * 4 and lib.prime_rms_norm_backward_scratch_bytes(-1, 64) < 0 and lib.prime_rms_norm_backward_scratch_bytes(1, 0) < 0

    def back(g=p, h=p, w=p, inv=p, rows=3, dim=64, t=0, wt=0, gx=p, gw=p, scratch=p, nbytes=need):
        return lib.prime_rms_norm_quantize_backward(g, 64, h, 64, w, inv, None, 0, rows, dim, t, wt, gx, gw, scratch, nbytes, None)

    for bad in (dict(g=None), dict(h=None), dict(w=None), dict(inv=None), dict(gx=None), dict(gw=None), dict(rows=-1), dict(dim=0), dict(t=4), dict(wt=2)):
        assert back(**bad) == -1, bad
    assert back(scratch=None) == -2 and back(nbytes=need - 1) == -2 and back(scratch=ctypes.c_void_p(4098)) == -2

    def quant(w=p, n=3, k=64, t=0, g=64, st=0, packed=p, scales=p):
        return lib.prime_quantize_4bit(w, 64, n, k, t, g, st, packed, scales, None)

    assert quant(n=0, w=None) == 0
    for bad in (dict(w=None), dict(packed=None), dict(scales=None), dict(n=-1), dict(k=0), dict(t=3), dict(g=16), dict(g=96), dict(st=2)):
        assert quant(**bad) == -1, bad

    def deq(packed=p, scales=p, n=3, k=64, g=64, st=0, out=p, ot=0):
        return lib.prime_dequantize_4bit(packed, 32, scales, 1, n, k, g, st, out, ot, None)

    assert deq(n=0, out=None) == 0
    for bad in (dict(packed=None), dict(scales=None), dict(out=None), dict(n=-1), dict(k=0), dict(ot=3), dict(g=0), dict(st=1 << 8)):
        assert deq(**bad) == -1, bad

    def mv(x=p, xt=0, xs=None, packed=p, scales=p, rows=2, n=3, k=64, g=64, st=0, out=p, ot=0):
        return lib.prime_matvec_4bit(x, 64, xt, xs, packed, 32, scales, 1, rows, n, k, g, st, out, ot, None)

    assert mv(rows=0, x=None) == 0 and mv(n=0, out=None) == 0
    for bad in (dict(x=None), dict(packed=None), dict(scales=None), dict(out=None), dict(xt=4), dict(xt=3), dict(xs=p), dict(rows=-1), dict(n=-1), dict(k=0),
                dict(g=33), dict(st=2), dict(ot=3), dict(n=(1 << 26) + 1)):
        assert mv(**bad) == -1, bad
    # rows of codes or scales 4 GiB apart
    assert lib.prime_matvec_4bit(p, 64, 0, None, p, 1 << 32, p, 1, 2, 3, 64, 64, 0, p, 0, None) == -1
    assert lib.prime_matvec_4bit(p, 64, 0, None, p, 32, p, 1 << 30, 2, 3, 64, 64, 0, p, 0, None) == -1


def test_reference_rounds_to_e4m3_as_the_type_is_defined():
    # every e4m3 number is its own nearest; midpoints go to the even neighbour
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64)
    fine = every[torch.isfinite(every)]
    assert torch.equal(ref.e4m3(fine), fine)
    v = torch.unique(fine[fine >= 0])
    mid = (v[1:] + v[:-1]) / 2
    even = torch.where(torch.arange(len(mid)) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(ref.e4m3(mid), even) and torch.equal(ref.e4m3(mid * (1 + 2.0 ** -40)), v[1:]) and torch.equal(ref.e4m3(mid * (1 - 2.0 ** -40)), v[:-1])


def test_reference_packing_is_its_own_inverse():
    codes = torch.randint(-8, 8, (3, 64), dtype=torch.int8)
    assert torch.equal(ref.unpack(ref.pack(codes)), codes)
    assert int(ref.pack(torch.tensor([[1, -1]], dtype=torch.int8))[0, 0]) == 0xF1


@pytest.mark.parametrize("frozen, thawed", [((0,), ()), ((2,), ()), ((), (3,)), ((0,), (3,))], ids=["first", "last", "one more", "another one"])
def test_outer_weights_are_refused_for_a_changed_set_of_parameters(frozen, thawed):
    from prime_amd.diloco import Diloco

    model = torch.nn.Sequential(*(torch.nn.Linear(64, 64, bias=False) for _ in range(4)))
    model[3].weight.requires_grad_(False)
    state = Diloco(0.7, model)
    for i in frozen:
        model[i].weight.requires_grad_(False)
    for i in thawed:
        model[i].weight.requires_grad_(True)
    with pytest.raises(RuntimeError, match="model does not match"):
        state.outer_weights_4bit(model)


def test_outer_weights_come_under_their_own_names(monkeypatch):
    from prime_amd.diloco import Diloco

    monkeypatch.setattr(lowbit, "quantize_4bit", lambda w, group, dtype: (w.clone(), None))
    model = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.LayerNorm(64), torch.nn.Linear(64, 64, bias=False))
    state = Diloco(0.7, model)
    want = {"0.weight": model[0].weight.detach().clone(), "2.weight": model[2].weight.detach().clone()}
    for p in model.parameters():
        p.data.add_(1.0)
    for wrapped, prefix in ((model, ""), (torch.compile(model, backend="eager"), "_orig_mod.")):
        got = state.outer_weights_4bit(wrapped)
        assert got.keys() == {prefix + n for n in want}
        assert all(torch.equal(got[prefix + n][0], w) for n, w in want.items())


def test_only_eager_calls_pass_the_dispatcher_by():
    """Whatever has to see an op (a compiler, a tracer, a mode, a transform) is noticed, though its tensors are plain by their type."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = {}

    def look(name):
        def f(t):
            seen[name] = lowbit._eager()
            return t * 2
        return f

    x = torch.randn(2, 3)
    look("plain")(x)
    with torch.no_grad():
        look("no_grad")(x)
    make_fx(look("make_fx"))(x)
    torch.vmap(look("vmap"))(x)
    torch.func.grad(lambda t: look("grad")(t).sum())(x)
    torch.func.jvp(look("jvp"), (x,), (x,))
    torch.jit.trace(look("trace"), x, check_trace=False)
    with forward_ad.dual_level():
        look("dual")(forward_ad.make_dual(x, x))

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Mode():
        look("mode")(x)
    look("plain again")(x)
    assert seen == {"plain": True, "no_grad": True, "make_fx": False, "vmap": False, "grad": False, "jvp": False, "trace": False, "dual": False,
                    "mode": False, "plain again": True}
    compiled = torch.compile(lambda t: t + 1 if lowbit._eager() else t - 1, backend="eager", fullgraph=True)
    assert torch.equal(compiled(x), x - 1)


def _ops_of(fn, *args):
    """The ops in the one graph that ``fn`` is compiled to (which is not run)."""
    names = []

    def backend(gm, inputs):
        names.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function" and "prime_lowbit" in str(n.target))
        outputs = [n for n in gm.graph.nodes if n.op == "output"][0].args[0]
        return lambda *a: tuple(torch.zeros(n.meta["example_value"].shape, dtype=n.meta["example_value"].dtype) for n in outputs)

    torch._dynamo.reset()
    torch.compile(fn, backend=backend, fullgraph=True)(*args)
    return names


def test_every_function_compiles_to_its_op_in_one_graph():
    x, w, inv = torch.randn(3, 64), torch.ones(64), torch.ones(3)
    packed, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1)
    for name, fn, args in (("rms_norm_quantize", lambda a, b: lowbit.rms_norm_quantize(a, b), (x, w)),
                           ("add_rms_norm_quantize", lambda a, b: lowbit.add_rms_norm_quantize(a, a, b, 1e-5, torch.float8_e4m3fn), (x, w)),
                           ("rms_norm_quantize_backward", lambda a, b, c: lowbit.rms_norm_quantize_backward(a, a, b, c), (x, w, inv)),
                           ("quantize_4bit", lambda a: lowbit.quantize_4bit(a, 32), (x,)),
                           ("dequantize_4bit", lambda a, b: lowbit.dequantize_4bit(a, b, 60), (packed, s)),
                           ("matvec_4bit", lambda a, b, c: lowbit.matvec_4bit(a, b, c), (x, packed, s))):
        ops = _ops_of(fn, *args)
        assert len(ops) == 1 and name in ops[0], (name, ops)


def test_gradients_are_refused_by_the_dispatcher_in_both_modes():
    from torch.autograd import forward_ad

    x, w = torch.randn(3, 64, device="meta"), torch.ones(64, device="meta")
    packed, s = torch.zeros(4, 32, dtype=torch.uint8, device="meta"), torch.ones(4, 1, device="meta")
    calls = (lambda t: lowbit.rms_norm_quantize(t, w), lambda t: lowbit.add_rms_norm_quantize(x, t, w),
             lambda t: lowbit.rms_norm_quantize_backward(t, x, w, torch.ones(3, device="meta")), lambda t: lowbit.quantize_4bit(t, 64),
             lambda t: lowbit.matvec_4bit(t, packed, s), lambda t: lowbit.dequantize_4bit(packed, t[:, :1].repeat(2, 1)[:4].contiguous()))
    for call in calls:
        call(x)
        with torch.no_grad():
            call(x.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="no gradient"):
            call(x.clone().requires_grad_())
        with forward_ad.dual_level():
            call(x)
            with pytest.raises(RuntimeError, match="no gradient"):
                call(forward_ad.make_dual(x, x))
        for transform in (lambda: torch.func.grad(lambda t: torch.utils._pytree.tree_leaves(call(t))[-1].float().sum())(x), lambda: torch.func.jvp(call, (x,), (x,))):
            with pytest.raises(RuntimeError, match="no gradient"):
                transform()


@pytest.mark.parametrize("case", range(len(_refusals())))
def test_what_a_call_refuses_its_trace_refuses(case):
    """The shape-only implementations make the checks of the ones that launch: a graph is not made of calls that cannot run."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    what, call, args = _refusals()[case]
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        args = tuple(mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args)
        with pytest.raises(RuntimeError, match=what):
            getattr(torch.ops.prime_lowbit, call.__name__[1:])(*args)


def test_tensors_on_two_devices_are_refused_in_a_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(3, 64, device="meta"), torch.empty(64)
        packed, s = torch.empty(4, 32, dtype=torch.uint8, device="meta"), torch.empty(4, 1)
        for call in (lambda: lowbit.rms_norm_quantize(x, w), lambda: lowbit.dequantize_4bit(packed, s), lambda: lowbit.matvec_4bit(x, packed, s)):
            with pytest.raises(RuntimeError, match="device"):
                call()


@pytest.mark.parametrize("n, k, group", [(48, 20000, 128), (15, 5604, 32), (60, 6000, 64), (20, 4300, 128)])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float16, torch.float32])
def test_the_bound_of_products_notices_lost_columns(n, k, group, xt):
    # 128 columns left out, or one column met with its neighbour's code, of a reference that is otherwise exact
    g = torch.Generator().manual_seed(n * k)
    codes = torch.randint(-8, 8, (n, -(-k // group) * group), generator=g, dtype=torch.int8)
    s = 0.01 * torch.exp(0.5 * torch.randn(n, codes.shape[1] // group, generator=g))
    x = (torch.randn(3, k, generator=g) * torch.exp(0.3 * torch.randn(k, generator=g))).to(xt)
    want, bound = ref.matvec(x, None, codes, s, k)[0], ref.matvec_bound(x, codes, s, k)
    assert ref.outside(want.float(), want, bound) <= 0
    for first in range(0, k, 128):
        less = x.clone()
        less[:, first:first + 128] = 0
        assert ref.outside(ref.matvec(less, None, codes, s, k)[0].float(), want, bound) > 0
    column = int((x[0, :-1].abs().float()).argmax())
    wrong = codes.clone()
    wrong[:, column] = codes[:, column + 1]
    assert ref.outside(ref.matvec(x, None, wrong, s, k)[0].float(), want, bound) > 0


def test_c_abi_refuses_scales_so_far_apart_that_their_bytes_leave_64_bits():
    from prime_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)
    for stride in (1 << 30, 1 << 32, 1 << 61, 1 << 62, (1 << 63) - 1):
        assert lib.prime_matvec_4bit(p, 64, 0, None, p, 32, p, stride, 2, 3, 64, 64, 0, p, 0, None) == -1, stride


def test_outer_weights_of_a_data_parallel_model(monkeypatch):
    from prime_amd.diloco import Diloco

    monkeypatch.setattr(lowbit, "quantize_4bit", lambda w, group, dtype: (w.clone(), None))
    model = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.Linear(32, 64))
    wrapped = torch.nn.DataParallel(model)
    for built, given, prefix in ((model, wrapped, "module."), (wrapped, model, ""), (wrapped, torch.compile(wrapped, backend="eager"), "_orig_mod.module.")):
        got = Diloco(0.7, built).outer_weights_4bit(given)
        assert {n: torch.equal(w, model.get_parameter(n[len(prefix):])) for n, (w, _) in got.items()} == {prefix + "0.weight": True, prefix + "1.weight": True}
