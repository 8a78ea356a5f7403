"""The library does not depend on the extension module over torch's tensors:
it is built first, and a failure there is reported and passed over.  The
module is built again for another torch or Python (no compiler needed: the
commands are stand-ins)."""
import os
import subprocess

import pytest

from ssla_rt_b200 import build


@pytest.fixture
def parts(monkeypatch, tmp_path):
    """build's outputs under tmp_path; run: the commands' outputs, in order."""
    run = []
    for name, path in (("LIB", "lib.so"), ("S01G_LIB", "s01g.so"), ("OPS_TORCH", "ops.so"), ("CONSUMER_CUBIN", "c.cubin"),
                       ("OPS_TORCH_STAMP", "_build/stamp")):
        monkeypatch.setattr(build, name, str(tmp_path / path))

    def command(cmd, check):
        out = cmd[cmd.index("-o") + 1]
        if run_fails in out:
            raise subprocess.CalledProcessError(1, cmd)
        open(out, "w").close()
        run.append(os.path.basename(out))

    run_fails = "\0"

    def fail(name):
        nonlocal run_fails
        run_fails = name

    monkeypatch.setattr(build.subprocess, "run", command)
    return run, fail


def test_the_library_comes_before_the_module(parts):
    run, _ = parts
    assert build.build() == build.LIB
    assert run == ["c.cubin", "lib.so", "ops.so"]
    build.build()
    assert run == ["c.cubin", "lib.so", "ops.so"]      # nothing is built twice


def test_the_library_is_built_where_the_module_is_not(parts, capsys):
    run, fail = parts
    fail("ops.so")
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert run == ["c.cubin", "lib.so"] and "without their extension module" in capsys.readouterr().err


def test_the_library_is_built_without_torch(parts, monkeypatch, capsys):
    run, _ = parts

    def no_torch():
        raise ImportError("No module named 'torch'")
    monkeypatch.setattr(build, "ops_torch_abi", no_torch)
    assert build.build() == build.LIB and run == ["c.cubin", "lib.so"]
    assert "No module named" in capsys.readouterr().err


def test_a_failing_library_is_an_error(parts):
    _, fail = parts
    fail("lib.so")
    with pytest.raises(subprocess.CalledProcessError):
        build.build()


def test_the_module_is_built_again_for_another_torch(parts, monkeypatch):
    run, fail = parts
    build.build()
    monkeypatch.setattr(build, "ops_torch_abi", lambda: "torch 0.0 python other")
    build.build()
    assert run[3:] == ["ops.so"]
    monkeypatch.setattr(build, "ops_torch_abi", lambda: "torch 0.1 python other")
    fail("ops.so")
    build.build()
    assert not os.path.exists(build.OPS_TORCH)            # rather than one that does not fit
