"""The language-model operators on the emulator build of the kernels, and the library's own refusal to run without a GPU."""
import os

import pytest
import torch

import lm_checks


@pytest.mark.parametrize('name', [n for n, _, where in lm_checks.CHECKS if where in ('both', 'cpu')])
def test_lm(name, emu_lib):
    fn = next(f for n, f, _ in lm_checks.CHECKS if n == name)
    fn(lm_checks.Env('cpu', emu_lib))


def test_product_library_refuses_without_a_gpu():
    """no CPU path: the library that is shipped answers JPPGPU_NO_DEVICE (4), the torch layer refuses CPU tensors"""
    import __graft_entry__ as ge
    from jumanpp_amd import lm
    if not os.path.exists(ge.LIB) or torch.cuda.is_available():
        pytest.skip('needs the built library and no GPU')
    lib = lm._lib(ge.LIB)
    t, out, ids = torch.zeros(4, 8), torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    assert lib.jppgpu_lm_embed(lm._rows(t, 't'), 4, 8, lm._ids(ids), 2, 1.0, lm._rows(out, 'out'), 0, None) == 4
    assert b'no HIP device' in lib.jppgpu_last_error()
    with pytest.raises(lm.JppGpuError):
        lm.embed(t, ids)
