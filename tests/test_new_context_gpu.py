"""Every kernel runs in a second CUDA context of the same device as in the first."""

import json
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = pathlib.Path(__file__).resolve().parent


def test_calls_in_a_second_context():
    out = subprocess.run([sys.executable, str(HERE / "new_context_child.py")], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    got = json.loads(out.stdout.strip().splitlines()[-1])
    for codes in got["codes"]:
        assert codes == [0] * 18
    assert all(got["some"]) and all(map(all, got["same"]))
