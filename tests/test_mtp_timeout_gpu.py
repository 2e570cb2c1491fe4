"""A bounded device wait that runs out inside an MTP call fails that call, not
the next pass, and leaves the host's and the device's positions together.
With IQ_QMV_TEST_TIMEOUT one weight copy is never requested, and the wait for
it ends after a short bound (test_timeout_gpu.py says why no GPU fault, trap
or hang is involved).  Runs in a child process so that the knob stays there."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = r"""
import numpy as np
from inferq_b200 import image, synth
from inferq_b200._lib import IqError
from inferq_b200.model import Model, State
cfg = synth.mini_35b()
m = Model(cfg, list(synth.generate(cfg, seed=1)))
hid = np.random.default_rng(0).standard_normal((4, cfg.hidden_size)).astype(np.float32)
for kv in ("f32", "i8"):
    st = State(m, 256, kv=kv)
    st.import_image(image.synthetic(cfg, 40, seed=1))
    def call(name, f):
        try:
            f()
            print(kv, name, "NO-ERROR", st.position, st.mtp_position)
        except IqError as e:
            print(kv, name, e.code, st.position, st.mtp_position)
    call("sync", lambda: st.mtp_sync(30, hid[0], [1, 2, 3], hid[:3]))
    call("draft", lambda: st.mtp_draft(1, hid[0], 3, cfg.vocab_size))
    before = st.position
    call("verify", lambda: st.verify([1, 2]))
    print(kv, "moved", st.position - before)
"""


def test_mtp_calls_report_their_own_waits(cuda):
    env = dict(os.environ, IQ_QMV_TEST_TIMEOUT="1")
    r = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [l.split() for l in r.stdout.splitlines()]
    for kv, got in (("f32", lines[:4]), ("i8", lines[4:])):
        assert got[0] == [kv, "sync", "-6", "40", "30"], got
        assert got[1] == [kv, "draft", "-6", "40", "30"], got
        assert got[2][:3] == [kv, "verify", "-6"] and got[3][2] in ("1", "2"), got  # the seed row at least is committed
