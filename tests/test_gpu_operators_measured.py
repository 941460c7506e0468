"""perf/operators.py: the calls that it makes of the library, next to its plain
forms on the same inputs, in a process of their own (torch brings a HIP
runtime, which has to be there before the library's).

Outputs are laid out alike.  Whole numbers are equal; stored rows differ by a
rounding of their type at most (both sides round once: a step, eps); f32
results by the sums' roundings, relative to the whole output (1e-5, over 100
roundings at the sums' lengths here)."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import sys
import torch
from perf import operators as o

def leaves(x, at=""):
    if isinstance(x, dict):
        return [l for k in x for l in leaves(x[k], at + "." + k)]
    return [(at, x)]

cases = []
for i, dt in enumerate(("f32", "f16", "bf16")):
    for tree in (False, True):
        cases.append(dict(kind="rope", b=9, nh=16, nkv=8, pos0=70, dtype=dt, tree=tree))
    cases.append(dict(kind="tree", b=9 + 20 * i, ctx=700, nh=16, nkv=8, dtype=dt))
    cases.append(dict(kind="window", b=1 + 70 * i, ctx=900, window=256, sinks=4, nh=16, nkv=8, dtype=dt))
    cases.append(dict(kind="copy", bufs=4, nkv=2, slots=90, n=40, pos0=7, src_rows=50, dtype=dt))
    cases.append(dict(kind="logprobs", rows=3, vocab=30011, k=(0, 5, 64)[i], dtype=dt))
for c in cases:
    print(c, flush=True)
    out = []
    for own in (False, True):
        o.own = own
        st = o.prepare(c, 5)
        o.run(st)
        out.append([(n, t.clone()) for n, t in leaves(o.run(st))])
    torch.cuda.synchronize()
    assert [n for n, _ in out[0]] == [n for n, _ in out[1]]
    for (n, a), (_, b) in zip(*out):
        assert a.shape == b.shape and a.dtype == b.dtype, n
        if not a.dtype.is_floating_point:
            assert torch.equal(a, b), n
            continue
        a, b, eps = a.double(), b.double(), 1e-5 if a.dtype == torch.float32 else torch.finfo(a.dtype).eps
        assert (a - b).norm() <= eps * a.norm(), (n, float((a - b).norm() / a.norm()))
print("done")
"""


def test_calls_and_plain_forms(gpu):
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout[-400:] + r.stderr[-2000:]
