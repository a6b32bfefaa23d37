"""The developer tools that rebuild the library's sources keep up with them."""
import os

import __graft_entry__ as ge

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_sanitizer_pass_has_every_unit_and_the_language_model_checks(tmp_path):
    """tools/emu_asan.sh: what it builds has the entry points of both headers, what it runs the checks of both"""
    text = open(os.path.join(ROOT, 'tools', 'emu_asan.sh')).read()
    units = [os.path.basename(src) for src, _ in ge._units()]
    assert 'jppgpu_lm.cc' in units
    assert 'build_emu_variant(' in text or all(u in text for u in units)
    assert 'tests/test_lm_cpu.py' in text and 'tests/test_cpu_parity.py' in text
