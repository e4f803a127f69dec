"""What the native calls behind rotary positions, whole-prompt attention, token weights and eviction do around a launch, with the
launches, the allocator and the devices replaced: tensors on the host's memory that say they lie on some GPU, and a record
of the device that each launch met and of what it was given.  csrc/window_bind.cpp is compiled here against those, so no GPU is needed."""

import importlib.util
import subprocess
import sysconfig
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="replaces the GPUs of this process")

STUB = r"""
#include "window_bind.cpp"

#include <ATen/ops/from_blob.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/utils/pybind.h>

#include <vector>

namespace {
int current = 0;
std::vector<std::vector<int64_t>> launches;   // the current device at each, and some of its arguments

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
// (Another test of this process may have put its own in place; its devices do as well.)
const bool registered = [] {
  try {
    c10::impl::getDeviceGuardImpl(at::kCUDA)->getDevice();
  } catch (...) {  // the real one, which finds no device here
    c10::impl::DeviceGuardImplRegistrar(at::kCUDA, new Devices());
  }
  return true;
}();
int met() { return c10::impl::getDeviceGuardImpl(at::kCUDA)->getDevice().index(); }

Tensor on(at::IntArrayRef size, ScalarType type, int device) {
  int64_t n = 1;
  for (int64_t s : size) n *= s;
  void* p = aligned_alloc(64, (n + 1) * 64);   // kept: a test's few
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
size_t hck_kv4_page_bytes(int dim) { return (size_t)dim * 136; }
int hck_rotary(const void*, int size, int64_t tokens, const uint64_t*, int rotated, int, int, float, int, int dim, const void*,
               int64_t, int64_t, int heads, void*, const void*, int64_t, int64_t, int kv, void*, void*) {
  launches.push_back({met(), size, tokens, rotated, dim, heads, kv});
  return 0;
}
size_t hck_prompt_attend_workspace_bytes(int64_t, int, int, int, int, int, int) { return 64; }
int hck_prompt_attend(const void*, const void*, const void*, int, int64_t tokens, int heads, int group, int dim, int64_t, int64_t,
                      int64_t, int64_t, int64_t, int64_t, const int32_t* starts, int seqs, int most, int, double, void*, float*, float*,
                      float*, void* work, size_t bytes, void*) {
  launches.push_back({met(), tokens, heads, group, dim, starts != nullptr, seqs, most, work != nullptr, (int64_t)bytes});
  return 0;
}
size_t hck_kv4_weigh_workspace_bytes(int64_t, int, int, int, int, int) { return 64; }
int hck_kv4_weigh(const void*, int64_t, int, int, int, const void*, int64_t, int group, int64_t, int64_t, const int32_t*, int64_t,
                  int cols, const int32_t*, const int32_t* starts, int seqs, int most, int, double, const float*, const float* prior,
                  int64_t, int64_t, int places, float*, void* work, size_t bytes, void*) {
  launches.push_back({met(), group, cols, starts != nullptr, seqs, most, prior != nullptr, places, work != nullptr, (int64_t)bytes});
  return 0;
}
size_t hck_kv4_evict_workspace_bytes(int, int, int) { return 64; }
int hck_kv4_evict(void*, int64_t, int, int, const int32_t*, int64_t, int cols, const int32_t*, int seqs, const float*, int64_t, int64_t,
                  int places, const int32_t*, int64_t, int into, int keep, int recent, int32_t*, int32_t*, float*, void* work, size_t bytes,
                  void*) {
  launches.push_back({met(), cols, seqs, places, into, keep, recent, work != nullptr, (int64_t)bytes});
  return 0;
}
}

PYBIND11_MODULE(_window_stub, m) {
  m.def("on", [](std::vector<int64_t> size, at::Tensor like, int device) { return on(size, like.scalar_type(), device); });
  m.def("current", [] { return met(); });
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
    for name in ("_window_stub", "_window"):
        spec = importlib.util.spec_from_file_location(name, so)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        modules.append(module)
    return modules


def inputs(stub, device):
    def on(size, dtype):
        return stub[0].on(size, torch.zeros(0, dtype=dtype), device)

    pool = (on([4, 2, 128 * 136], torch.uint8), 4, 2, 128, device)
    return dict(pool=pool, turns=on([64], torch.int64), at=on([3], torch.int64), q=on([3, 4, 128], torch.bfloat16),
                kv=on([3, 2, 128], torch.bfloat16), table=on([3, 5], torch.int32), lengths=on([3], torch.int32),
                starts=on([4], torch.int32), lse=on([3, 4], torch.float32), weights=on([3, 2, 300], torch.float32),
                into=on([3, 2], torch.int32))


def calls(stub, x):
    w = stub[1]
    return [lambda: w.rotate(x["turns"], 128, 128, False, 1.0, x["at"], x["q"], x["kv"], False),
            lambda: w.prompt(x["q"], x["kv"], x["kv"], x["starts"], 2, True, None, True),
            lambda: w.weigh(*x["pool"], x["q"], x["table"], x["lengths"], x["lse"], x["starts"], 2, True, None, x["weights"]),
            lambda: w.evict(*x["pool"], x["table"], x["lengths"], x["weights"], x["into"], 200, 7)]


@pytest.mark.parametrize("device", [0, 2])
def test_each_call_launches_on_its_tensors_device(stub, device):
    want = [[8, 3, 128, 128, 4, 2], [3, 2, 2, 128, 1, 3, 2, 1, 64], [2, 5, 1, 3, 2, 1, 300, 1, 64], [5, 3, 300, 2, 200, 7, 1, 64]]
    for call, arguments in zip(calls(stub, inputs(stub, device)), want):
        got = call()
        assert stub[0].launches() == [[device, *arguments]]
        assert stub[0].current() == 0      # the caller's device is as it was
        for t in got if isinstance(got, tuple) else (got,):
            assert t.device == torch.device("cuda", device)


def test_tensors_of_two_devices_are_refused(stub):
    x = inputs(stub, 1)
    other = inputs(stub, 2)
    for name, which in (("at", (0,)), ("kv", (0, 1)), ("q", (0, 1, 2)), ("starts", (1, 2)), ("table", (2, 3)), ("lengths", (2, 3)),
                        ("lse", (2,)), ("weights", (2, 3)), ("into", (3,))):
        mixed = calls(stub, {**x, name: other[name]})
        for i in which:
            with pytest.raises(ValueError):
                mixed[i]()
    assert not stub[0].launches()


def test_the_pools_bytes_are_asked_for_at_each_call(stub):
    x = inputs(stub, 1)
    like = torch.zeros(0, dtype=torch.uint8)
    for bad in (stub[0].on([4, 2, 128 * 136 - 1], like, 1), stub[0].on([4, 2, 128 * 136], like, 0), x["pool"][0][:3]):
        for call in calls(stub, {**x, "pool": (bad, *x["pool"][1:])})[2:]:
            with pytest.raises(ValueError, match="buf"):
                call()
    assert not stub[0].launches()


def test_what_is_left_out(stub):
    """Without keys, starts, prior: none reach the launch; a prior of no places is none."""
    x, w = inputs(stub, 0), stub[1]
    assert w.rotate(x["turns"], 128, 64, False, 1.0, x["at"], x["q"], None, True).shape == (3, 4, 128)
    assert stub[0].launches() == [[0, 8, 3, 64, 128, 4, 0]]
    got = w.prompt(x["q"], x["kv"], x["kv"], None, None, True, None, False)
    assert got[2] is None and got[3] is None and stub[0].launches() == [[0, 3, 2, 2, 128, 0, 1, 3, 1, 64]]
    for prior in (None, x["weights"][..., :0]):
        w.weigh(*x["pool"], x["q"], x["table"], x["lengths"], x["lse"], None, None, True, None, prior)
        assert stub[0].launches() == [[0, 2, 5, 0, 3, 1, 0, 0, 1, 64]]
