"""The 4-bit cache's ops and torch's dispatcher: the registered ops do what the functions of ``ops`` do, and a
call of those functions is seen by whatever looks on from the dispatcher, as the bf16 ops' are."""

from __future__ import annotations

import pytest
import torch
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from solort_b200 import ops

BF, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8
NAMES = ["qk_norm_rope_append_int4", "kv_store_int4", "kv_load_int4", "gqa_decode_paged_int4"]
NH, NKV, P, T = 8, 2, 16, 5


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name.removeprefix("solort_attn::"))
        return func(*args, **(kwargs or {}))


class SeenFunctions(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func).removeprefix("solort_attn."))
        return func(*args, **(kwargs or {}))


class Counted(torch.Tensor):
    """A subclass that notes the ops it takes part in."""

    names: list[str] = []

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        Counted.names.append(func._schema.name.removeprefix("solort_attn::"))
        args, kwargs = torch.utils._pytree.tree_map_only(
            Counted, lambda t: t.inner, (args, kwargs or {}))
        return func(*args, **kwargs)


def counted(t: torch.Tensor) -> Counted:
    c = torch.Tensor._make_wrapper_subclass(Counted, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)
    c.inner = t
    return c


def state(device="cuda"):
    g = torch.Generator(device).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=device).to(BF)  # noqa: E731
    return {"qkv": r(T, (NH + 2 * NKV) * 128), "qn": r(128), "kn": r(128), "cos": r(64, 128), "sin": r(64, 128),
            "positions": torch.arange(T, device=device), "slots": torch.arange(7, 7 + T, device=device),
            "pages": ops.kv_pages_int4(4, NKV, P, device=device), "q_out": torch.zeros(T, NH, 128, dtype=BF, device=device),
            "key": r(T, NKV, 128), "value": r(T, NKV, 128), "q": r(2, 1, NH, 128),
            "table": torch.tensor([[0, 1], [1, 2]], dtype=I32, device=device),
            "q_pos": torch.tensor([9, 20], device=device), "out": torch.zeros(2, 1, NH, 128, dtype=BF, device=device),
            "workspace": torch.zeros(1 << 22, dtype=U8, device=device),
            "q_lens": torch.ones(2, dtype=I32, device=device)}


def call(name: str, s: dict):
    """One call through ``ops``; what it wrote."""
    if name == "qk_norm_rope_append_int4":
        ops.qk_norm_rope_append_int4(s["qkv"], s["qn"], s["kn"], 1e-6, s["cos"], s["sin"], s["positions"], s["slots"],
                                     s["pages"], num_qo_heads=NH, num_kv_heads=NKV, q_out=s["q_out"])
        return s["pages"], s["q_out"]
    if name == "kv_store_int4":
        ops.kv_store_int4(s["key"], s["value"], s["slots"], s["pages"])
        return (s["pages"],)
    if name == "kv_load_int4":
        return ops.kv_load_int4(s["pages"], s["slots"], key=s["key"], value=s["value"])
    ops.gqa_decode_paged_int4(s["q"], s["pages"], s["table"], s["q_pos"], max_kv_len=32, out=s["out"],
                              workspace=s["workspace"], q_lens=s["q_lens"])
    return (s["out"],)


def registered(name: str, s: dict):
    """The same through ``torch.ops``."""
    o = torch.ops.solort_attn
    if name == "qk_norm_rope_append_int4":
        o.qk_norm_rope_append_int4(s["qkv"], s["qn"], s["kn"], 1e-6, s["cos"], s["sin"], s["positions"], s["slots"],
                                   s["pages"], s["q_out"])
        return s["pages"], s["q_out"]
    if name == "kv_store_int4":
        o.kv_store_int4(s["key"], s["value"], s["slots"], s["pages"])
        return (s["pages"],)
    if name == "kv_load_int4":
        o.kv_load_int4(s["pages"], s["slots"], s["key"], s["value"])
        return s["key"], s["value"]
    o.gqa_decode_paged_int4(s["q"], s["pages"], s["table"], s["q_pos"], s["out"], s["workspace"], 32, None, s["q_lens"])
    return (s["out"],)


def filled(s: dict) -> dict:
    ops.kv_store_int4(torch.randn(64, NKV, 128, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(BF),
                      torch.randn(64, NKV, 128, generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(BF),
                      torch.arange(64, device="cuda"), s["pages"])
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_the_registered_op_does_what_the_function_does(name):
    for a, b in zip(call(name, filled(state())), registered(name, filled(state()))):
        assert torch.equal(a, b) and a.any()
    assert ops.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_the_call(name):
    s, want = filled(state()), call(name, filled(state()))
    with Seen() as mode:
        got = call(name, s)
    assert mode.names == [name]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_function_mode_sees_the_call(name):
    s = filled(state())
    with SeenFunctions() as mode:
        call(name, s)
    assert name in mode.names


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_a_trace_of_real_tensors_has_the_call(name, pre_dispatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    s = filled(state())
    keys = sorted(s)
    graph = make_fx(lambda *t: call(name, dict(zip(keys, t))), pre_dispatch=pre_dispatch)(*[s[k] for k in keys])
    assert [n.target._schema.name for n in graph.graph.nodes if n.op == "call_function"
            and "solort_attn" in n.target._schema.name] == [f"solort_attn::{name}"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_profile_names_the_call(name):
    s = filled(state())
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        call(name, s)
    assert f"solort_attn::{name}" in [e.key for e in prof.key_averages()]


@pytest.mark.gpu
@pytest.mark.parametrize("name,field", [("qk_norm_rope_append_int4", "qkv"), ("qk_norm_rope_append_int4", "kn"),
                                        ("kv_store_int4", "value"), ("kv_load_int4", "slots"),
                                        ("gqa_decode_paged_int4", "q"), ("gqa_decode_paged_int4", "q_lens")])
def test_a_subclass_among_the_tensors_sees_the_call(name, field):
    s, want = filled(state()), call(name, filled(state()))
    s[field] = counted(s[field])
    Counted.names = []
    got = call(name, s)
    assert Counted.names == [name]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_parameters_and_inference_mode(name):
    """Weights as a module holds them, and a call in inference mode."""
    want, s = call(name, filled(state())), filled(state())
    for k in ("qn", "kn"):
        s[k] = torch.nn.Parameter(s[k])
    with torch.inference_mode():
        got = call(name, s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_compiled_function_has_the_call(name):
    s, want, found = filled(state()), call(name, filled(state())), []

    def backend(module, inputs):
        found.extend(str(n.target) for n in module.graph.nodes if n.op == "call_function")
        return module

    got = torch.compile(lambda t: call(name, t), backend=backend, fullgraph=True)(s)
    assert [f for f in found if "solort_attn" in f or "int4" in f] != []
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_plain_calls_alone_may_pass_the_dispatcher_by(monkeypatch):
    """Without a GPU: what the functions of ``ops`` decide from, with a tensor that says it is on one."""

    class OnDevice:
        is_cuda = True

    on, t = OnDevice(), torch.zeros(1)
    monkeypatch.setattr(ops, "_PLAIN_TYPES", ops._PLAIN_TYPES | {OnDevice})
    assert ops._direct(on, t, None, torch.nn.Parameter(t)) and not ops._direct(t, t)
    with torch.inference_mode(), torch.no_grad():
        assert ops._direct(on, t)
    with Seen():
        assert not ops._direct(on, t)
    with SeenFunctions():
        assert not ops._direct(on, t)
    with torch.autograd.profiler.profile():
        assert not ops._direct(on, t)
    with torch._subclasses.FakeTensorMode():
        assert not ops._direct(on, t)
    assert not ops._direct(on, counted(t))
    inside = []
    torch.vmap(lambda x: (inside.append(ops._direct(on, t)), x)[1])(torch.ones(2))
    torch.jit.trace(lambda x: (inside.append(ops._direct(on, t)), x + 1)[1], torch.ones(2), check_trace=False)
    assert inside and not any(inside) and ops._direct(on, t)
