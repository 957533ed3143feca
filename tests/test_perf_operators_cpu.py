"""The measured operators' file: its framework calls find the package wherever the program was started, every op it calls is
there, and the package can be imported from the root of a checkout as it is."""
import ast
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILE = os.path.join(REPO, "perf", "operators.py")


def run(code, cwd):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    r = subprocess.run([sys.executable, "-c", code, FILE], cwd=cwd, env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


@pytest.mark.parametrize("where", ["root", "elsewhere"])
def test_the_framework_is_found(where, tmp_path):
    """A fresh process that knows nothing of the package's place loads the file and resolves every op it calls."""
    with open(FILE) as f:
        tree = ast.parse(f.read())
    called = sorted({n.func.attr for n in ast.walk(tree) if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute)
                     and isinstance(n.func.value, ast.Name) and n.func.value.id == "ops"})
    assert len(called) >= 6
    out = run("import importlib.util, sys\n"
              "spec = importlib.util.spec_from_file_location('cases', sys.argv[1])\n"
              "M = importlib.util.module_from_spec(spec)\n"
              "spec.loader.exec_module(M)\n"
              "ops = M._ops()\n"
              f"print(sum(callable(getattr(ops, n)) for n in {called!r}))\n", REPO if where == "root" else str(tmp_path))
    assert int(out) == len(called)


def test_the_package_is_importable_from_the_root():
    out = run("from vllm_xpu_kernels import ops, cabi\nprint(callable(ops.fp8_block_scaled_mm), cabi.lib().kvc_version() > 0)", REPO)
    assert out.split() == ["True", "True"]
