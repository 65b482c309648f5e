// The Python function that times a call while a recorder is active (timing.timed).
#pragma once

#include <pybind11/pybind11.h>

#include <atomic>
#include <utility>

namespace cl {

// Calls come from any thread, without the GIL, and so while the block that records ends: the hook
// is only tested there.  It is changed and borrowed under the GIL; a thread that waited for the
// GIL may find it gone, and its call then runs untimed.
class TimedHook {
    std::atomic<PyObject*> hook_{nullptr};  // owned

  public:
    // Under the GIL; None: no recorder.
    void set(pybind11::object timed) {
        PyObject* next = timed.is_none() ? nullptr : timed.release().ptr();
        Py_XDECREF(hook_.exchange(next));
    }

    template <typename F>
    void run(const char* name, F&& call) {
        if (hook_.load(std::memory_order_relaxed)) {
            pybind11::gil_scoped_acquire gil;
            const auto timed = pybind11::reinterpret_borrow<pybind11::object>(hook_.load());
            if (timed) {
                timed(name, pybind11::cpp_function(std::forward<F>(call)));
                return;
            }
        }
        call();
    }
};

}  // namespace cl
