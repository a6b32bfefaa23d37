"""tests/lm_checks.py as a program: what it leaves when a check fails."""
import json

import torch

import lm_checks


def fake(monkeypatch, *checks):
    monkeypatch.setattr(lm_checks, 'CHECKS', [(name, fn, 'both') for name, fn in checks])
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda: None)


def bad(text):
    def check(E):
        raise RuntimeError(text)
    return check


def test_a_failed_gpu_leaves_its_trace_and_ends_the_run(monkeypatch, tmp_path):
    fake(monkeypatch, ('fine', lambda E: None), ('faults', bad('HIP error: of a kind')), ('never', lambda E: None))
    path = tmp_path / 'results.json'
    lm_checks.run_all('cpu', None, str(path))
    done = json.load(open(path))
    assert done['fine'] == 'ok' and 'HIP error: of a kind' in done['faults'] and 'never' not in done


def test_status_without_a_results_file(monkeypatch, capsys):
    fake(monkeypatch, ('fine', lambda E: None))
    assert lm_checks.main([], 'cpu') == 0
    fake(monkeypatch, ('fine', lambda E: None), ('wrong', bad('no')), ('fine too', lambda E: None))
    assert lm_checks.main([], 'cpu') == 1
    assert '3 checks, 1 failed' in capsys.readouterr().out
    fake(monkeypatch, ('faults', bad('HIP error')), ('never', lambda E: None))
    assert lm_checks.main([], 'cpu') == 1
    assert '1 of 2 checks' in capsys.readouterr().out


def test_status_with_one_is_the_readers(monkeypatch, tmp_path):
    """a reader of the results has every check's own: the status says that they are there"""
    fake(monkeypatch, ('fine', lambda E: None), ('wrong', bad('no')))
    path = tmp_path / 'results.json'
    assert lm_checks.main([str(path)], 'cpu') == 0
    assert set(json.load(open(path))) == {'fine', 'wrong'}


def test_names_are_unique():
    names = [n for n, _, _ in lm_checks.CHECKS]
    assert len(set(names)) == len(names)
