"""The XLA FFI handlers of the dense products and of the gradients' clipping: operands of other
lengths, ranks and dtypes than the first one's imply are refused, since the C ABI takes them as
pointers alone. Compiled against a stub of XLA's API and called on the host. Against XLA itself:
parity unpinned."""

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_operands_of_other_lengths_and_dtypes_are_refused(tmp_path):
    exe = tmp_path / "handlers"
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(HERE, "xla_stub"),
                    "-I", os.path.join(os.path.dirname(HERE), "include"), "-I", "/opt/rocm/include",
                    os.path.join(HERE, "xla_handlers_dense.cc"), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    handlers = {}
    for at, line in enumerate(lines):
        what, taken, calls, right = line.rsplit(" ", 3)
        assert calls == taken and right == "1", (at, line)
        handlers.setdefault(what, []).append(taken)
    assert set(handlers) == {"rows", "units backward", "contract", "slope", "clip"}
    assert all({"0", "1"} == set(v) for v in handlers.values())
