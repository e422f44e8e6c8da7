"""perf/operators.py hands torch's memory to the library, whose stream is not torch's: what prepare returns has to be written,
and a pass that is waited for afterwards has the right result.  In a process of its own: torch brings a HIP runtime along,
which has to be loaded before the library is."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT
from tests.gpu_util import say

pytestmark = pytest.mark.gpu

PROGRAM = '''
import importlib.util, sys
import torch
sys.path.insert(0, '.')
spec = importlib.util.spec_from_file_location('operator_cases', 'perf/operators.py')
m = importlib.util.module_from_spec(spec)
spec.loader.exec_module(m)
for c in m.listed():
    print('prepare', c['name'], flush=True)
    s = m.prepare(c, 3)
    assert torch.cuda.current_stream().query(), "work on the inputs is still queued on torch's stream"
    if c['kind'] == 'keep8':
        m.own = True
        got = m.run(s)
        from litenn_amd.core.hip import api
        api.synchronize(0)
        assert torch.equal(got, m._kept_values(*m._codes(s['x']), c['n']))
    torch.cuda.synchronize()
print('all written')
'''


def test_prepared_inputs_are_written(hip):
    say('prepare of every listed case')
    r = subprocess.run([sys.executable, '-u', '-c', PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and 'all written' in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
