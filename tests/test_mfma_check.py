"""The check that the build makes of matrix instructions written as asm (csrc/check_mfma.py), on made-up assembly."""
import importlib.util
import os

from conftest import ROOT

spec = importlib.util.spec_from_file_location('check_mfma', os.path.join(ROOT, 'he-cka-ensembles_amd', 'csrc', 'check_mfma.py'))
check_mfma = importlib.util.module_from_spec(spec)
spec.loader.exec_module(check_mfma)

MFMA = '\t;;#ASMSTART\n\tv_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]\n\t;;#ASMEND\n'


def faults(*lines):
    body = ''.join(l if l.endswith('\n') else '\t%s\n' % l for l in lines)
    return check_mfma.check('\n_Z6kernelv: ; @_Z6kernelv\n%s\ts_endpgm\n\t.section\n' % body)


def test_an_operand_just_written_is_found():
    for between, bad in ((['s_nop 1'], 0), (['s_nop 0'], 1), ([], 1), (['s_waitcnt lgkmcnt(0)', 's_mov_b32 s0, 0'], 0)):
        seen, found = faults('v_mov_b32_e32 v9, v1', *between, MFMA)
        assert seen == 1 and len(found) == bad, (between, found)
    assert faults('ds_read_b128 v[8:11], v1', MFMA) == (1, [])          # not a vector instruction: waited for by a counter
    assert len(faults('v_accvgpr_write_b32 a2, 0', MFMA)[1]) == 1


def test_a_sum_read_too_early_is_found():
    for between, bad in (([], 1), (['s_nop 15'], 1), (['s_nop 15', 's_nop 15'], 0)):
        assert len(faults(MFMA, *between, 'v_accvgpr_read_b32 v20, a1')[1]) == bad
    assert faults(MFMA, 'v_accvgpr_read_b32 v20, a9') == (1, [])
    assert faults(MFMA, MFMA) == (2, [])
    assert len(faults(MFMA, 'scratch_store_dwordx4 off, a[0:3], s0')[1]) == 1
