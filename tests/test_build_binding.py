"""_torch_ops.so is rebuilt for another interpreter or PyTorch (make -n: nothing is built here)."""
import os
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "manifold_b200", "csrc")


def _plan(python):
    """What make would run for the binding, with the library's objects taken as built."""
    res = subprocess.run(["make", "-n", "-C", CSRC, "../_torch_ops.so", f"PYTHON={python}"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return res.stdout


def _other(tmp_path, old, new):
    """An interpreter that answers as this one, but for one value."""
    path = tmp_path / "python"
    path.write_text(f"#!/bin/sh\nexec {sys.executable} -c \"import sysconfig, importlib.metadata as _m\n{old} = {new}\n$2\"\n")
    path.chmod(0o755)
    return str(path)


def test_the_binding_is_up_to_date_for_this_interpreter():
    subprocess.run(["make", "-C", CSRC, "../_torch_ops.so", f"PYTHON={sys.executable}"], check=True, capture_output=True)
    assert "torch_ops.cpp" not in _plan(sys.executable)


def test_another_abi_or_pytorch_rebuilds_the_binding(tmp_path):
    subprocess.run(["make", "-C", CSRC, "../_torch_ops.so", f"PYTHON={sys.executable}"], check=True, capture_output=True)
    for old, new in (("_m.version", "lambda name: '0.0.other'"),
                     ("sysconfig.get_config_var", "lambda name: 'cpython-399-other'")):
        assert "torch_ops.cpp" in _plan(_other(tmp_path, old, new)), old
    assert "torch_ops.cpp" not in _plan(sys.executable)  # nothing was touched
