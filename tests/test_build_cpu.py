"""How the extension is linked."""

import ast
import glob
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _link_flags():
    for node in ast.walk(ast.parse(open(os.path.join(ROOT, "setup.py")).read())):
        if isinstance(node, ast.Assign) and getattr(node.targets[0], "id", "") == "LINK_FLAGS":
            return ast.literal_eval(node.value)
        if isinstance(node, ast.keyword) and node.arg == "extra_link_args" and isinstance(node.value, ast.List):
            return ast.literal_eval(node.value)
    raise AssertionError("setup.py names no link flags")


def test_link_flags_are_the_linkers():
    """Only what every compiler hands on to its linker: driver flags such as -nostdlib++ need a new enough one."""

    assert all(flag.startswith(("-l", "-L", "-Wl,")) for flag in _link_flags())


def test_extension_shares_the_cpp_runtime():
    """The runtime is a dependency, and no second copy of its locale is inside."""

    libs = glob.glob(os.path.join(ROOT, "representax_b200", "_C*.so"))
    if not libs or shutil.which("readelf") is None or shutil.which("nm") is None:
        pytest.skip("the extension is not built here, or binutils are missing")
    dynamic = subprocess.run(["readelf", "-d", libs[0]], capture_output=True, text=True, check=True).stdout
    assert "libstdc++.so.6" in dynamic
    symbols = subprocess.run(["nm", "-D", "--defined-only", libs[0]], capture_output=True, text=True, check=True).stdout
    assert "_ZNSt6locale" not in symbols
