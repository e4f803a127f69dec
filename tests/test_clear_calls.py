"""What the native calls behind holmes_amd.clear do around a launch, with the launches, the allocator and the devices
replaced: tensors on the host's memory that say they lie on some GPU, and a record of the device that each launch met.
csrc/clear_bind.cpp is compiled here against those, so no GPU is needed."""

import importlib.util
import subprocess
import sysconfig
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="replaces the GPUs of this process")

STUB = r"""
#include "clear_bind.cpp"

#include <ATen/ops/from_blob.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/utils/pybind.h>

#include <vector>

namespace {
int current = 0;
std::vector<int> launches;   // the current device at each

struct Devices final : c10::impl::DeviceGuardImplInterface {
  c10::DeviceType type() const override { return at::kCUDA; }
  c10::Device exchangeDevice(c10::Device d) const override {
    const int old = current;
    current = d.index();
    return c10::Device(at::kCUDA, (c10::DeviceIndex)old);
  }
  c10::Device getDevice() const override { return c10::Device(at::kCUDA, (c10::DeviceIndex)current); }
  void setDevice(c10::Device d) const override { current = d.index(); }
  void uncheckedSetDevice(c10::Device d) const noexcept override { current = d.index(); }
  c10::Stream getStream(c10::Device d) const override { return c10::Stream(c10::Stream::DEFAULT, d); }
  c10::Stream exchangeStream(c10::Stream s) const override { return s; }
  c10::DeviceIndex deviceCount() const noexcept override { return 4; }
};
C10_REGISTER_GUARD_IMPL(CUDA, Devices)

Tensor on(at::IntArrayRef size, ScalarType type, int device) {
  int64_t n = 1;
  for (int64_t s : size) n *= s;
  void* p = calloc(n + 1, 16);   // kept: a test's few
  const at::Device d(at::kCUDA, (at::DeviceIndex)device);
  return at::from_blob(p, size, [](void*) {}, at::TensorOptions().dtype(type).device(d), d);
}
}  // namespace

namespace at::detail {
TensorBase empty_cuda(IntArrayRef size, ScalarType type, std::optional<Device> d, std::optional<MemoryFormat>) {
  return on(size, type, d->index());
}
}  // namespace at::detail
namespace c10::hip {
HIPStream getCurrentHIPStream(DeviceIndex i) {
  return HIPStream(HIPStream::UNCHECKED, Stream(Stream::DEFAULT, Device(at::kCUDA, i)));
}
}  // namespace c10::hip

extern "C" {
int hck_kv4_append(void*, int64_t, int, int, int, const void*, int64_t, int64_t, const void*, int64_t, int64_t,
                   const int64_t*, int64_t, void*) { launches.push_back(current); return 0; }
int hck_kv4_read(const void*, int64_t, int, int, int, const int64_t*, int64_t, void*, void*, void*) {
  launches.push_back(current); return 0; }
size_t hck_kv4_page_bytes(int dim) { return (size_t)dim * 136; }
size_t hck_kv4_attend_workspace_bytes(int64_t, int, int, int, int, int, int) { return 64; }
int hck_kv4_attend(const void*, int64_t, int, int, int, const void*, int64_t, int, int64_t, int64_t, const int32_t*, int64_t,
                   int, const int32_t*, const int32_t*, int, int, int, float, void*, float*, float*, float*, void*, size_t,
                   void*) { launches.push_back(current); return 0; }
size_t hck_token_scores_workspace_bytes(int64_t, int, int, int) { return 64; }
int hck_token_scores(const void*, int, int64_t, int, int64_t, const int64_t*, int, float*, float*, int64_t*, float*, void*,
                     size_t, void*) { launches.push_back(current); return 0; }
}

PYBIND11_MODULE(_stub, m) {
  m.def("on", [](std::vector<int64_t> size, at::Tensor like, int device) { return on(size, like.scalar_type(), device); });
  m.def("current", [] { return current; });
  m.def("launches", [] { auto got = launches; launches.clear(); return got; });
}
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    from torch.utils import cpp_extension

    from holmes_amd import build

    at = tmp_path_factory.mktemp("stub")
    (at / "stub.cpp").write_text(STUB)
    so = at / "_stub.so"
    include = [*cpp_extension.include_paths(), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    done = subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-DUSE_ROCM",
                           "-D__HIP_PLATFORM_AMD__=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                           *(f"-isystem{p}" for p in include), f"-I{build.CSRC}", str(at / "stub.cpp"), "-o", str(so),
                           f"-L{Path(torch.__file__).parent / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip",
                           "-ltorch_python"], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]
    modules = []
    for name in ("_stub", "_clear"):
        spec = importlib.util.spec_from_file_location(name, so)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        modules.append(module)
    return modules


def inputs(stub, device):
    def on(size, dtype):
        return stub[0].on(size, torch.zeros(0, dtype=dtype), device)

    pool = (on([4, 2, 128 * 136], torch.uint8), 4, 2, 128, device)
    return dict(pool=pool, kv=on([3, 2, 128], torch.bfloat16), slots=on([3], torch.int64), table=on([3, 1], torch.int32),
                lengths=on([3], torch.int32), starts=on([4], torch.int32), logits=on([3, 10], torch.float32),
                tokens=on([3], torch.int64))


def calls(stub, x):
    c = stub[1]
    return [lambda: c.append(*x["pool"], x["kv"], x["kv"], x["slots"]),
            lambda: c.read(*x["pool"], x["slots"], torch.float32),
            lambda: c.attend(*x["pool"], x["kv"], x["table"], x["lengths"], x["starts"], 1, True, None, True),
            lambda: c.scores(x["logits"], x["tokens"], 4)]


@pytest.mark.parametrize("device", [0, 2])
def test_each_call_launches_on_its_tensors_device(stub, device):
    for call in calls(stub, inputs(stub, device)):
        got = call()
        assert stub[0].launches() == [device]
        assert stub[0].current() == 0      # the caller's device is as it was
        for t in got if isinstance(got, tuple) else ():
            assert t.device == torch.device("cuda", device)


def test_the_pools_bytes_are_asked_for_at_each_call(stub):
    """An address kept from the pool's making would outlive its tensor."""
    x = inputs(stub, 1)
    like = torch.zeros(0, dtype=torch.uint8)
    buf = x["pool"][0]
    for bad in (stub[0].on([4, 2, 128 * 136 - 1], like, 1), stub[0].on([4, 2, 128 * 136], like, 0), buf.transpose(0, 1),
                buf[:3], stub[0].on([4, 2, 128 * 136], torch.zeros(0), 1), torch.zeros((4, 2, 128 * 136), dtype=torch.uint8)):
        for call in calls(stub, {**x, "pool": (bad, *x["pool"][1:])})[:3]:
            with pytest.raises(ValueError, match="buf"):
                call()
    for call in calls(stub, {**x, "pool": (buf.data_ptr(), *x["pool"][1:])})[:3]:
        with pytest.raises(TypeError, match="buf"):
            call()
    assert stub[0].launches() == []


def test_inputs_that_require_a_gradient(stub):
    """Results without a graph would pass for constants: refused, but where gradients are off."""
    x = inputs(stub, 1)
    x["kv"].requires_grad_()
    x["logits"].requires_grad_()
    append, read, attend, scores = calls(stub, x)
    for call, name in ((append, "keys"), (attend, "queries"), (scores, "logits")):
        with pytest.raises(ValueError, match=f"{name} require a gradient"):
            call()
    assert stub[0].launches() == []
    with torch.no_grad():
        for call in (append, read, attend, scores):
            call()
    assert stub[0].launches() == [1] * 4


def test_strides_of_single_elements(stub):
    """One sequence's length out of a table of several numbers, one column out of wider tables."""
    x = inputs(stub, 0)
    one = torch.zeros(0, dtype=torch.int32)
    wide = stub[0].on([3, 4], one, 0)
    x["kv"], x["starts"] = x["kv"][:1], stub[0].on([2], one, 0)
    for lengths, table in ((wide[:1, 1], wide[:1]), (wide[:1, 0], wide[:1, ::4]), (wide[:1, 0], wide[:1].t()[:1].t())):
        assert lengths.stride(0) == 4
        stub[1].attend(*x["pool"], x["kv"], table, lengths, x["starts"], 1, True, None, False)
    none = stub[0].on([1], one, 0)
    stub[1].attend(*x["pool"], x["kv"][:0], wide[:0, ::2], wide[:0, 0], none, 0, True, None, False)
    assert stub[0].launches() == [0] * 4
    with pytest.raises(ValueError, match="contiguous"):
        stub[1].attend(*x["pool"], x["kv"], wide[:1, ::2], wide[:1, 0], x["starts"], 1, True, None, False)
