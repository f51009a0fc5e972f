"""A call whose launch fails says so, and the next call does not say it again."""

import json
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = pathlib.Path(__file__).resolve().parent


def test_an_error_is_reported_by_its_own_call_alone():
    out = subprocess.run([sys.executable, str(HERE / "failed_launch_child.py")], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    got = json.loads(out.stdout.strip().splitlines()[-1])
    assert set(got["refused"].values()) == {-6}, got["refused"]
    assert set(got["after"].values()) == {0}, got["after"]
