"""The PyTorch binding shares the C++ runtime of the process: what its code throws, numbers in the message and all, is a Python exception."""
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent
SOURCE = """
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
using namespace torch::autograd;
struct Node1 : Function<Node1> {
  static variable_list forward(AutogradContext*, const at::Tensor& x) { return {x * 2}; }
  static variable_list backward(AutogradContext*, variable_list g) {
    const int rc = (int)g.size() - 8;
    TORCH_CHECK(rc == 0, "a gradient: the library returned code ", rc);
    return g;
  }
};
PyObject* twice(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  return THPVariable_Wrap(Node1::apply(THPVariable_Unpack(o))[0]);
  END_HANDLE_TH_ERRORS
}
PyMethodDef methods[] = {{"twice", twice, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "small", nullptr, -1, methods};
PyMODINIT_FUNC PyInit_small() { return PyModule_Create(&module); }
"""
PROGRAM = """
import importlib.util, torch
spec = importlib.util.spec_from_file_location("small", {path!r})
small = importlib.util.module_from_spec(spec)
spec.loader.exec_module(small)
x = torch.ones(3, requires_grad=True)
try:
    small.twice(x).sum().backward()
except RuntimeError as e:
    assert "the library returned code -7" in str(e)
    print("raised")
"""


def test_an_error_with_a_number_in_it_is_raised(tmp_path):
    """Of a module that is built as the binding is, in a process of its own: with a runtime of the module's own it ended in a segmentation fault."""
    from workloadsuite_b200 import build

    source, out = tmp_path / "small.cpp", tmp_path / "small.so"
    source.write_text(SOURCE)
    keep, build.TORCH_LIB = build.TORCH_LIB, out
    try:
        job = build._start_torch_binding(torch, source)
    finally:
        build.TORCH_LIB = keep
    log, _ = job.communicate()
    assert job.returncode == 0, log
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(path=str(out))], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "raised" in r.stdout, (r.returncode, r.stderr[-2000:])


def test_a_subclass_without_memory_stays_what_it_is():
    """One that wraps another tensor has no numbers of its own that a kernel could read: nothing is made of it that looks as if it had."""
    from workloadsuite_b200.ssd import _plain

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return cls(torch.ones(3))

    class Sub(torch.Tensor):
        pass

    w = Wrapper(torch.ones(3))
    assert _plain(w) is w and _plain(None) is None
    t = torch.ones(3, requires_grad=True)
    assert _plain(t) is t
    s = torch.ones(3).as_subclass(Sub).requires_grad_(True)
    p = _plain(s)
    assert type(p) is torch.Tensor and p.data_ptr() == s.data_ptr() and type(torch.autograd.grad(p.sum(), [s])[0]) in (torch.Tensor, Sub)
