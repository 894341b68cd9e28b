"""CPU: what `make` builds with and without torch."""
import os
import subprocess
import sys

import pytest
import torch

from helpers import REPO

CSRC = os.path.join(REPO, "procgen_amd", "csrc")
VERSION = os.path.join(os.path.dirname(torch.__file__), "version.py")
WITH_ROCM = os.path.exists(os.path.join(os.path.dirname(torch.__file__), "include", "c10", "hip", "HIPStream.h"))


def plan(*args):
    return subprocess.run(["make", "-n", "-C", CSRC, *args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def test_the_library_is_built_where_there_is_no_torch(tmp_path):
    without = plan(f"BUILD={tmp_path}", f"PYTHON={sys.executable} -S")  # -S: no installed packages
    assert without.returncode == 0, without.stdout
    assert f"{tmp_path}/libenv.so" in without.stdout and f"{tmp_path}/bake_atlas" in without.stdout and "learner_torch" not in without.stdout
    nothing = plan(f"BUILD={tmp_path}", "PYTHON=/nowhere/python")
    assert nothing.returncode == 0 and f"{tmp_path}/libenv.so" in nothing.stdout and "learner_torch" not in nothing.stdout
    asked = plan(f"BUILD={tmp_path}", f"PYTHON={sys.executable} -S", f"{tmp_path}/learner_torch.so")
    assert asked.returncode != 0 and "torch" in asked.stdout


@pytest.mark.skipif(not WITH_ROCM, reason="torch without ROCm's headers")
def test_the_torch_side_is_built_with_the_installed_torch(tmp_path):
    fresh = plan(f"BUILD={tmp_path}", f"PYTHON={sys.executable}")
    assert fresh.returncode == 0 and "learner_torch.cpp" in fresh.stdout
    if os.path.exists(os.path.join(CSRC, "build", "learner_torch.so")):  # another torch than it was built with: built again
        assert "learner_torch.cpp" in plan("-W", VERSION, f"PYTHON={sys.executable}", "build/learner_torch.so").stdout


def test_operators_say_what_is_missing(tmp_path):
    code = f"""import sys; sys.path.insert(0, {REPO!r})
from procgen_amd import learner_ops
try:
    learner_ops._ext.advantages
except ImportError as e:
    assert "learner_torch.so" in str(e) and "make" in str(e), e
else:
    raise SystemExit("loaded from nowhere")"""
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PROCGEN_AMD_LIB_DIR": str(tmp_path)}, stderr=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.skipif(not os.path.exists(os.path.join(CSRC, "build", "learner_torch.so")), reason="learner_torch.so not built (run __graft_entry__.build())")
def test_host_threads_may_be_the_first_to_call():
    """all of them at once: each finds every operator"""
    code = f"""import sys, threading; sys.path.insert(0, {REPO!r}); sys.setswitchinterval(1e-6)
from procgen_amd import learner_ops
start, errors = threading.Barrier(16), []
def call():
    start.wait()
    try:
        learner_ops._ext.policy_loss
    except Exception as e:
        errors.append(e)
threads = [threading.Thread(target=call) for _ in range(16)]
for t in threads: t.start()
for t in threads: t.join()
raise SystemExit(repr(errors) if errors else 0)"""
    for _ in range(5):
        r = subprocess.run([sys.executable, "-c", code], stderr=subprocess.PIPE, text=True)
        assert r.returncode == 0, r.stderr[-300:]
