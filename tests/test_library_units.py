"""The library of the training path alone, as the integration notes build it: mmn_kernels.hip by itself."""
import os
import subprocess
import sys

import pytest

from multimodn_amd import build

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
from multimodn_amd import hip, sequence
lib = hip.load()
assert lib.mmn_source_hash().decode() == "unknown" and lib.mmn_version() == hip.VERSION
try:
    sequence.causal_conv(torch.zeros(1, 2, 3), torch.zeros(3, 4))
except hip.MmnError as e:
    assert "no sequence operators" in str(e), e
    print("refused")
"""


def test_the_training_path_alone_loads(tmp_path):
    obj = os.path.join(build.OBJ, "mmn_kernels.o")
    if not os.path.exists(obj):
        pytest.skip("the library was not compiled here")
    alone = str(tmp_path / "libmmn_hip.so")
    subprocess.run([build.hipcc_path(), "--offload-arch=gfx950", "-shared", "-fPIC", obj, "-o", alone], check=True)
    run = subprocess.run([sys.executable, "-c", PROGRAM], cwd=REPO, env={**os.environ, "MMN_LIB_PATH": alone}, capture_output=True, text=True)
    assert run.returncode == 0 and "refused" in run.stdout, run.stderr[-2000:]


def test_the_packages_library_says_what_it_was_built_from():
    assert build.built_hash() == build.source_hash()
