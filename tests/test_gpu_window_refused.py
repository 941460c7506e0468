"""A windowed attention that is refused (forced from the host:
CMF_WINDOW_ATTN_FAIL=1) is an error of the call that ran it, eager or captured,
and the model goes on where no window is in the way."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import numpy as np
import cmf_amd
from cmf_amd import synth
from cmf_amd.model import Model
cmf_amd.init(0)
cfg = dict(n_layers=2, hidden=256, n_heads=4, n_kv=2, head_dim=128, inter=512, vocab=4096, max_seq=2048, rope_theta=1e6,
           eps=1e-6)
m = Model(synth.accept_model(cfg))
ids = synth.ids(1, 100, cfg["vocab"])

def refused(what, fn):
    try:
        fn()
    except cmf_amd.CmfError as e:
        assert "windowed attention" in str(e), e
        return
    raise SystemExit(what + " went through")

m.prefill(ids)
plain = m.decode(8, spec=False)[0].tolist()
m.prefill(ids)
spec = m.decode(8, spec=True, k=4)[0].tolist()
m.set_window(40, 2)
refused("prefill", lambda: m.prefill(ids))
refused("score", lambda: m.score(ids, top_k=2))
m.prefill(ids[:30])  # (nothing out of the window yet)
m.set_window(8)
refused("forward_batch", lambda: m.forward_batch(ids[:4], 30))
refused("verify_step", lambda: m.verify_step(ids[:3], 30))
refused("decode", lambda: m.decode(12, spec=False))
refused("speculative decode", lambda: m.decode(30, spec=True, k=4))
refused("speculative decode once more", lambda: m.decode(30, spec=True, k=4))
m.set_window(0)
m.prefill(ids)
assert m.decode(8, spec=False)[0].tolist() == plain
m.prefill(ids)
assert m.decode(8, spec=True, k=4)[0].tolist() == spec
print("done")
"""


def test_calls_report_a_refused_attention(gpu):
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT, CMF_WINDOW_ATTN_FAIL="1"),
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout[-300:] + r.stderr[-1500:]
