"""CPU test of build.py: what is built again, and what is not."""
from __future__ import annotations

import importlib.util
import os
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent


@pytest.fixture()
def build(tmp_path, monkeypatch):
    """build.py over a tree of empty files, whose commands only write their output."""
    spec = importlib.util.spec_from_file_location("build_under_test", REPO / "muon_fusion_ascend950_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for name, at in (("PKG", "pkg"), ("CSRC", "pkg/csrc"), ("INCLUDE", "include"), ("BUILD", "pkg/_build")):
        (tmp_path / at).mkdir(parents=True, exist_ok=True)
        monkeypatch.setattr(module, name, tmp_path / at)
    for sources in (module.CU_SOURCES, module.OP_SOURCES):
        for name, headers in sources.items():
            for path in [module.CSRC / name] + [module.CSRC / h if h.endswith(".cuh") else module.INCLUDE / h for h in headers]:
                if tmp_path in path.parents:
                    path.touch()
                    os.utime(path, (1000, 1000))
    made = []

    def run(cmd):
        out = Path(cmd[cmd.index("-o") + 1])
        made.append(out.name)
        out.touch()

    monkeypatch.setattr(module, "_run", run)
    module.made = made
    return module


def built(build):
    build.made.clear()
    build.build_all()
    return set(build.made)


def test_everything_is_built_once(build):
    objects = {f"{name}.o" for sources in (build.CU_SOURCES, build.OP_SOURCES) for name in sources}
    assert built(build) == objects | {build.LIB_NAME, build.OP_NAME}
    assert built(build) == set()


def test_libraries_that_came_without_objects_are_kept(build):
    built(build)
    for obj in build.BUILD.iterdir():
        obj.unlink()
    assert built(build) == set()


def test_a_changed_source_is_compiled_and_linked(build):
    built(build)
    later = max(p.stat().st_mtime for p in build.PKG.iterdir()) + 10
    os.utime(build.CSRC / "route_experts_sm100.cu", (later, later))
    assert {"route_experts_sm100.cu.o", build.LIB_NAME} <= built(build)
    assert "distill_topk_sm100.cu.o" not in build.made
