"""The language-model operators on the MI355X through torch: tests/lm_checks.py in one child process (torch's HIP runtime has
to come before the library's, and this process's tests open the library first), its results one test each."""
import json
import os
import subprocess
import sys

import pytest

import lm_checks

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def results(gpu_lib, tmp_path_factory):
    path = tmp_path_factory.mktemp('lm') / 'results.json'
    log = tmp_path_factory.mktemp('lm') / 'log.txt'
    with open(log, 'w') as f:
        rc = subprocess.call([sys.executable, '-u', os.path.join(ROOT, 'tests', 'lm_checks.py'), str(path)], stdout=f, stderr=subprocess.STDOUT,
                             timeout=280)
    tail = open(log).read()[-2000:]
    done = json.load(open(path)) if os.path.exists(path) else {}
    return rc, done, tail


@pytest.mark.gpu
@pytest.mark.parametrize('name', [n for n, _, where in lm_checks.CHECKS if where in ('both', 'gpu')])
def test_gpu_lm(name, results):
    rc, done, tail = results
    assert name in done, 'the child process ended (rc %s) before this check:\n%s' % (rc, tail)
    assert done[name] == 'ok', done[name]
    assert rc == 0, tail
