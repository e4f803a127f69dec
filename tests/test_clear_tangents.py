"""Forward-mode derivatives through the cleartext operators, which have none: inputs with a tangent are refused.  On the stand-ins
for the GPUs of test_clear_calls and test_clear_window_calls, so no GPU is needed."""

import importlib.util
import subprocess
import sysconfig
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from holmes_amd import build

from . import test_clear_calls as cache
from . import test_clear_window_calls as window

pytestmark = window.pytestmark


def compiled(at, text, stub, calls):
    """The stand-ins and the calls of another test's source, the former as a module of another name (one of the same name would
    be the other test's)."""
    from torch.utils import cpp_extension

    name = stub + "_of_tangents"
    text = text.replace(f"PYBIND11_MODULE({stub},", f"PYBIND11_MODULE({name},")
    assert name in text
    (at / "stub.cpp").write_text(text)
    include = [*cpp_extension.include_paths(), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    done = subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-DUSE_ROCM",
                           "-D__HIP_PLATFORM_AMD__=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                           *(f"-isystem{p}" for p in include), f"-I{build.CSRC}", str(at / "stub.cpp"), "-o", str(at / "stub.so"),
                           f"-L{Path(torch.__file__).parent / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip",
                           "-ltorch_python"], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]
    modules = []
    for n in (name, calls):
        spec = importlib.util.spec_from_file_location(n, at / "stub.so")
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        modules.append(module)
    return modules


@pytest.fixture(scope="module")
def cache_stub(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("cache"), cache.STUB, "_stub", "_clear")


@pytest.fixture(scope="module")
def window_stub(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("window"), window.STUB, "_window_stub", "_window")


def refused(stub, module, x, name, which, argument):
    """Each of the calls is refused for x[name] with a tangent, and goes through with that tensor detached, without forward mode
    and behind the level."""
    like = x[name]
    tangent = stub[0].on(list(like.shape), torch.zeros(0, dtype=like.dtype), like.device.index)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(like, tangent)
        run = module.calls(stub, {**x, name: dual})
        for i in which:
            with pytest.raises(ValueError, match=f"{argument} have a tangent"):
                run[i]()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):   # which says nothing of forward mode
                run[i]()
        assert not stub[0].launches()
        plain = module.calls(stub, {**x, name: dual.detach()})
        for i in which:
            plain[i]()
            with forward_ad._set_fwd_grad_enabled(False):
                run[i]()
        assert len(stub[0].launches()) == 2 * len(which)
    for i in which:
        run[i]()
    assert len(stub[0].launches()) == len(which)


@pytest.mark.parametrize("name,which,argument", [("kv", (0,), "keys"), ("kv", (2,), "queries"), ("logits", (3,), "logits")])
def test_cache(cache_stub, name, which, argument):
    refused(cache_stub, cache, cache.inputs(cache_stub, 1), name, which, argument)


@pytest.mark.parametrize("name,which,argument", [("q", (0, 1, 2), "queries"), ("kv", (0, 1), "keys"), ("lse", (2,), "lse"),
                                                 ("weights", (2,), "prior"), ("weights", (3,), "weights")])
def test_window(window_stub, name, which, argument):
    refused(window_stub, window, window.inputs(window_stub, 1), name, which, argument)
