"""An edited source or header makes every binary that is built from it stale."""
import os
import subprocess

import pytest

import tdc_build as B


def _included(unit):
    """What the preprocessor opens for `unit`, of this repository's files."""
    torch_like = unit.endswith(".cpp")
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    incs = [f"-I{B.INCLUDE}", f"-I{B.CSRC}", f"-I{cuda}"]
    if torch_like:
        import sysconfig
        import torch.utils.cpp_extension as ce
        incs += [f"-I{i}" for i in ce.include_paths("cuda")] + [f"-I{sysconfig.get_paths()['include']}"]
    out = subprocess.run(["g++", "-M", "-x", "c++", "-std=c++17", *incs, os.path.join(B.CSRC, unit)],
                         capture_output=True, text=True, check=True).stdout
    names = out.replace("\\\n", " ").split()[1:]
    return {os.path.realpath(n) for n in names if os.path.realpath(n).startswith(B.REPO + os.sep)}


@pytest.mark.parametrize("unit", [*B.UNITS, *B.EXT_SOURCES])
def test_dependencies_are_what_the_compiler_opens(unit):
    assert {os.path.realpath(p) for p in B._deps(unit)} == _included(unit)


def test_an_edited_header_makes_its_units_stale(tmp_path):
    # a target as new as its newest source is up to date; a second behind any one it is not
    for unit in (*B.UNITS, *B.EXT_SOURCES):
        deps = B._deps(unit)
        target = tmp_path / (unit + ".o")
        target.write_text("")
        for d in deps:
            os.utime(target, (0, os.path.getmtime(d) - 1))
            assert B._stale(str(target), [d]), d
        os.utime(target, (0, max(map(os.path.getmtime, deps))))
        assert not B._stale(str(target), deps)
    assert any(p.endswith("tdc_delta_grad.cuh") for p in B._deps("tdc_sequence.cu"))
