"""CPU check: the sizes of the whole-matrix operators' workspaces depend on
the arguments alone.  A program may ask for a size while another device is
current than the one it then calls on; the size has to do there too.

The library asks for a device's SM count through glmb::sm_count(), which is
replaced here by a preloaded one that answers with a given number."""
import json
import os
import subprocess
import sys

import pytest

from gpu_algos_b200 import capi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SIZES = [(nf, nt, ntasks) for nf, nt in ((33, 33), (40, 5000), (256, 4096), (4096, 4096), (777, 1000), (333, 1021))
         for ntasks in (1, 3, 40, 1000, 65535)]
PREDICT = [(4096, 16384, 1, 2048, 128), (2901, 5003, 1, 17, 64), (256, 16, 64, 500, 64)]

ASK = """
import json, sys
from gpu_algos_b200 import capi
L = capi.lib()
sizes, predict = json.loads(sys.argv[1])
print(json.dumps([getattr(L, f"glmm_orthogonal_workspace_size_{s}")(*a) for s in capi.MATRIX for a in sizes]
                 + [getattr(L, f"glmm_predict_q4_workspace_size_{s}")(*a) for s in capi.MATRIX for a in predict]))
"""


@pytest.fixture(scope="module")
def fake_sm_count(tmp_path_factory):
    d = tmp_path_factory.mktemp("sm_count")
    src, lib = d / "sm_count.cpp", d / "libsm_count.so"
    src.write_text('#include <cstdlib>\nnamespace glmb { int sm_count() { return std::atoi(std::getenv("SM_COUNT")); } }\n')
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", str(src), "-o", str(lib)], check=True)
    return str(lib)


def test_workspace_sizes_do_not_depend_on_the_current_device(fake_sm_count):
    answers = []
    for sms in (8, 74, 148, 160):
        env = dict(os.environ, LD_PRELOAD=fake_sm_count, SM_COUNT=str(sms), PYTHONPATH=REPO)
        out = subprocess.run([sys.executable, "-c", ASK, json.dumps([SIZES, PREDICT])], env=env, cwd=REPO, check=True,
                             capture_output=True, text=True).stdout
        answers.append(json.loads(out))
    assert len(answers[0]) == len(capi.MATRIX) * (len(SIZES) + len(PREDICT)) and all(v > 0 for v in answers[0])
    assert all(a == answers[0] for a in answers)
