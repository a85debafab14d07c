"""The build notices a change in every header that a source includes."""
import importlib.util
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1] / "sm120-norm-fusion-kernels_b200"
spec = importlib.util.spec_from_file_location("package_build", ROOT / "build.py")
build = importlib.util.module_from_spec(spec)
spec.loader.exec_module(build)


def included(source: Path) -> set[Path]:
    """Headers of this repository that `source` includes, directly or not."""
    found, todo = set(), [source]
    while todo:
        for name in re.findall(r'^\s*#include "([^"]+)"', todo.pop().read_text(), re.M):
            for path in (build.CSRC / name, build.INCLUDE / name):
                if path.exists() and path not in found:
                    found.add(path)
                    todo.append(path)
    return found


@pytest.mark.parametrize("name", build.BINDING_SOURCES)
def test_binding_headers(name):
    assert included(build.CSRC / name) <= set(build._binding_headers())


@pytest.mark.parametrize("name", sorted({*build.NORM_SOURCES, *build.SERVING_SOURCES}))
def test_kernel_headers(name):
    assert included(build.CSRC / name) <= set(build._headers())
