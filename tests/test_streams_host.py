"""scp_amd/streams.py, host logic (no GPU)"""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("mode", ["overlap", "serial"])
def test_the_texture_stream_is_refused(mode):
    """SCP_TEXTURE_STREAM=1 asked for a third side stream, with which the device stops; it is an error, before anything runs"""
    env = dict(os.environ, SCP_TEXTURE_STREAM="1", SCP_STREAMS=mode, PYTHONPATH=os.path.join(ROOT, "self-corr-pose_amd"))
    r = subprocess.run([sys.executable, "-c", "import scp_amd.streams"], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode != 0 and "SCP_TEXTURE_STREAM" in r.stderr.splitlines()[-1], r.stderr
    env["SCP_TEXTURE_STREAM"] = "0"
    r = subprocess.run([sys.executable, "-c", "import scp_amd.streams"], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


def test_no_code_opens_a_texture_stream():
    """the step has two side streams: nothing but the refusal names a third"""
    pkg = os.path.join(ROOT, "self-corr-pose_amd", "scp_amd")
    for f in sorted(os.listdir(pkg)):
        if f.endswith(".py"):
            text = open(os.path.join(pkg, f)).read()
            assert "_tex_stream" not in text and "overlap_texture" not in text, f
