"""Every XLA FFI handler's binding names what its function takes: XLA's own registration does not
compile otherwise, and with it none of the handlers. Compiled on the host against a stub of XLA's
API whose registration checks that (tests/xla_bindings). Against XLA itself: parity unpinned."""

import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCE = os.path.join(ROOT, "bux_amd", "xla", "xla_ffi.cc")


def _compile(path):
    return subprocess.run(
        ["g++", "-std=c++17", "-fsyntax-only", "-D__HIP_PLATFORM_AMD__",
         "-I", os.path.join(HERE, "xla_bindings"), "-I", os.path.join(ROOT, "include"),
         "-I", "/opt/rocm/include", str(path)], capture_output=True, text=True)


def test_every_binding_is_its_handlers():
    done = _compile(SOURCE)
    assert done.returncode == 0, re.findall(r"error: .*", done.stderr)


@pytest.mark.parametrize("right, wrong", [
    (".Arg<In>().Attr<float>(\"a\").Ret<In>()", ".Arg<In>().Attr<float>(\"a\").Ret<In>().Ret<In>()"),
    (".Arg<In>().Attr<float>(\"a\").Ret<In>()", ".Arg<In>().Arg<In>().Attr<float>(\"a\").Ret<In>()"),
    (".Arg<In>().Attr<float>(\"a\").Ret<In>()", ".Arg<In>().Attr<int64_t>(\"a\").Ret<In>()"),
    (".Arg<In>().Attr<float>(\"a\").Ret<In>()", ".Attr<float>(\"a\").Arg<In>().Ret<In>()"),
], ids=["a result", "an operand", "an attribute's type", "the order"])
def test_a_binding_of_something_else_does_not_compile(tmp_path, right, wrong):
    for binding, compiles in ((right, True), (wrong, False)):
        path = tmp_path / "handler.cc"
        path.write_text(f"""
#include <hip/hip_runtime.h>
#include "xla/ffi/api/ffi.h"
namespace ffi = xla::ffi;
using In = ffi::AnyBuffer;
static ffi::Error H(hipStream_t, In, float, ffi::Result<In>) {{ return ffi::Error::Success(); }}
XLA_FFI_DEFINE_HANDLER_SYMBOL(
    BuxH, H, ffi::Ffi::Bind().Ctx<ffi::PlatformStream<hipStream_t>>(){binding});
""")
        done = _compile(path)
        assert (done.returncode == 0) == compiles, done.stderr
        assert compiles or "the binding is not its handler's" in done.stderr
