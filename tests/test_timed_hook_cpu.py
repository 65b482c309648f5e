"""The hook by which the C++ autograd Functions time their calls, driven from a small module of its
own: no device is needed, and a crash stays in the child process."""
import subprocess
import sys
import sysconfig
import textwrap

import pytest

from compactlogic_amd import build

SOURCE = r"""
#include "timed_hook.h"

#include <chrono>
#include <stdexcept>
#include <thread>

namespace py = pybind11;
static cl::TimedHook hook;

// This thread holds the GIL while another one makes a call, which therefore waits for the GIL to
// time itself; meanwhile the hook becomes `next`.
static bool changed_under_a_waiting_call(py::object next) {
    std::atomic<bool> ran{false};
    std::thread other([&] { hook.run("waited", [&] { ran = true; }); });
    std::this_thread::sleep_for(std::chrono::milliseconds(200));
    const bool waited = !ran;
    hook.set(std::move(next));
    {
        py::gil_scoped_release unlocked;
        other.join();
    }
    return waited && ran;
}

PYBIND11_MODULE(hooked, m) {
    m.def("set", [](py::object timed) { hook.set(std::move(timed)); });
    m.def("run", [] {
        int runs = 0;
        hook.run("call", [&] { ++runs; });
        return runs;
    }, py::call_guard<py::gil_scoped_release>());
    m.def("fail", [] { hook.run("fails", [] { throw std::out_of_range("failed"); }); },
          py::call_guard<py::gil_scoped_release>());
    m.def("changed_under_a_waiting_call", &changed_under_a_waiting_call);
}
"""


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from torch.utils.cpp_extension import include_paths
    at = tmp_path_factory.mktemp("hooked")
    (at / "hooked.cpp").write_text(SOURCE)
    dirs = [*include_paths(), sysconfig.get_paths()["include"]]
    subprocess.run([build._cxx(), "-O1", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                    "-pthread", f"-I{build.CSRC}", *(a for d in dirs for a in ("-isystem", d)),
                    str(at / "hooked.cpp"), "-o", str(at / "hooked.so")], check=True)
    return at


def _child(folder, code):
    return subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=folder, timeout=60,
                          capture_output=True, text=True)


def test_a_recorder_that_ends_while_a_call_waits(folder):
    got = _child(folder, """
        import hooked
        hooked.set(lambda name, fn: fn())
        assert hooked.changed_under_a_waiting_call(None)
        assert hooked.run() == 1
    """)
    assert got.returncode == 0, (got.returncode, got.stderr)


def test_a_recorder_that_changes_while_a_call_waits(folder):
    got = _child(folder, """
        import hooked
        seen = []
        hooked.set(lambda name, fn: seen.append("first"))
        assert hooked.changed_under_a_waiting_call(lambda name, fn: (seen.append(name), fn()))
        assert seen == ["waited"]
    """)
    assert got.returncode == 0, (got.returncode, got.stderr)


def test_calls_with_and_without_a_recorder(folder):
    """The hook gets the name and the call, may call it more than once or end itself meanwhile;
    what the call throws comes through it."""
    got = _child(folder, """
        import hooked
        seen = []

        def timed(name, fn):
            hooked.set(None)
            fn()
            fn()
            seen.append(name)

        assert hooked.run() == 1 and not seen
        hooked.set(timed)
        del timed
        assert hooked.run() == 2 and seen == ["call"]
        assert hooked.run() == 1 and seen == ["call"]
        for recorder in (None, lambda name, fn: fn()):
            hooked.set(recorder)
            try:
                hooked.fail()
            except IndexError as e:
                assert "failed" in str(e)
            else:
                raise AssertionError
    """)
    assert got.returncode == 0, (got.returncode, got.stderr)
