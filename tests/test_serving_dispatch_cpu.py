"""Whoever looks on at PyTorch's operators sees the serving operators: dispatch and
function modes, tensor subclasses in any argument, function transforms. (The
functions go past the dispatcher otherwise.)"""
import pytest
import torch
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from sm120_rmsnorm import extensions, serving

X = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
I = torch.zeros(2, dtype=torch.int32)
ARGS = {
    "plan_step_": [I, I, I[None], I, I[:1], 16, I, I, I.long(), I],
    "release_blocks_": [I, I.bool(), I[None], I, I[:1], 16],
    "prompt_attention": [X, X, X, X, I],
    "paged_decode_attention": [X, X, X[None], X[None], I[None], I],
    "qk_norm_mrope_cache_": [X, X, None, X[0, 0], X[0, 0], I.long()[None], X[0].float(), [64]],
}
FUNCTIONS = {name: getattr(serving, name, None) or getattr(extensions, name) for name in ARGS}


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())


class SeenFunctions(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        if hasattr(func, "name") and callable(func.name):
            self.names.append(func.name())
            return None
        return func(*args, **(kwargs or {}))


class Wrapped(torch.Tensor):
    seen = []

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(func.name())


@pytest.mark.parametrize("name", ARGS)
@pytest.mark.parametrize("mode", [Seen, SeenFunctions])
def test_modes(name, mode):
    with mode() as seen:
        FUNCTIONS[name](*ARGS[name])
    assert seen.names == [f"sm120_norm_ext::{name}"]


@pytest.mark.parametrize("name", ARGS)
def test_subclasses_in_any_argument(name):
    for i, arg in enumerate(ARGS[name]):
        if not isinstance(arg, torch.Tensor):
            continue
        args = list(ARGS[name])
        args[i] = arg.as_subclass(Wrapped)
        Wrapped.seen.clear()
        FUNCTIONS[name](*args)
        assert Wrapped.seen == [f"sm120_norm_ext::{name}"], i


def test_function_transforms_meet_the_registered_operator():
    def call(x):
        serving.prompt_attention(x, x, x, x, I)
        return x

    with pytest.raises((RuntimeError, NotImplementedError), match="sm120_norm_ext"):
        torch.vmap(call)(X[None])


def test_ordinary_calls_go_to_the_extension(monkeypatch):
    called = []

    class Extension:
        nothing_looks_on = staticmethod(serving._C.nothing_looks_on)

        def __getattr__(self, name):
            return lambda *args: called.append(name)

    monkeypatch.setattr(serving, "_extension", lambda: Extension())
    for name, function in FUNCTIONS.items():
        args = [torch.nn.Parameter(a, requires_grad=False) if a is X else a for a in ARGS[name]]
        function(*args)
    assert called == list(ARGS)
