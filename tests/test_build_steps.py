"""CPU-only: build() names the step that failed and the first error of it, and a clean tree's steps need no order
between them that make does not know."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

sys.path.insert(0, ROOT)
import __graft_entry__ as entry  # noqa: E402


def test_a_failing_step_is_named_with_its_first_error(tmp_path, monkeypatch):
    (tmp_path / "x").mkdir()
    (tmp_path / "x" / "Makefile").write_text("all:\n\t@echo 'a.hip:3:1: warning: w'\n\t@echo 'a.hip:7:2: error: first' >&2\n\t@echo 'a.hip:9:2: error: second'\n\t@exit 3\n")
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    with pytest.raises(RuntimeError, match=r"the library failed \(make -C x all: exit status 2\): a.hip:7:2: error: first"):
        entry._make("the library", "x", "all")
    (tmp_path / "x" / "Makefile").write_text("all:\n\t@echo fine\n")
    entry._make("the library", "x", "all")


@pytest.mark.parametrize("failing", [None, "thrust_amd/csrc", "oracle", "tests/cpp", "tests/emu"])
def test_build_fails_with_the_library_and_reports_the_programs_of_the_tests(monkeypatch, capsys, failing):
    ran = []

    def make(step, where, *args):
        ran.append(where)
        if where == failing:
            raise RuntimeError(f"build: {step} failed")
    monkeypatch.setattr(entry, "_make", make)
    if failing == "thrust_amd/csrc":
        with pytest.raises(RuntimeError, match="the library failed"):
            entry.build()
        return
    assert entry.build().__name__ == "thrust_amd"
    assert ran[0] == "thrust_amd/csrc" and {"oracle", "tests/cpp", "tests/emu"} <= set(ran)
    assert ("failed" in capsys.readouterr().err) == (failing is not None)


@pytest.mark.parametrize("where,target", [("tests/emu", "build/emu.o"), ("tests/emu", "build/lm_types.h"), ("tests/emu", "build/runtime.cpp"),
                                          ("thrust_amd/csrc", "build/runtime.o"), ("tests/cpp", "build/test_sort")])
def test_every_rule_makes_the_folder_that_it_writes_to(where, target):
    """In a clean tree any of them may be the first that runs."""
    plan = subprocess.run(["make", "-C", os.path.join(ROOT, where), "-n", "-B", target], capture_output=True, text=True)
    assert plan.returncode == 0, plan.stderr[-2000:]
    made = False
    for line in plan.stdout.splitlines():
        made = made or line.startswith("mkdir -p build")
        assert made or target not in line.split(), line
