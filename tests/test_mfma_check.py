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


LOOP = '.LBB0_1:\n'
AGAIN = 's_cbranch_scc1 .LBB0_1'


def test_the_way_back_to_a_loops_start_is_looked_at():
    assert len(faults(LOOP, MFMA, 's_add_i32 s0, s0, 1', 'v_mov_b32_e32 v9, v1', AGAIN)[1]) == 1      # two slots behind it: the branch is one
    assert faults(LOOP, MFMA, 'v_mov_b32_e32 v9, v1', 's_nop 0', AGAIN) == (1, [])
    assert len(faults(LOOP, 'v_accvgpr_read_b32 v20, a1', MFMA, AGAIN)[1]) == 1                       # a sum of the turn before
    assert faults(LOOP, 'v_accvgpr_read_b32 v20, a1', MFMA, 's_nop 15', AGAIN) == (1, [])
    # over a block that is jumped over, and past one that always leaves
    assert len(faults('v_mov_b32_e32 v9, v1', 's_cbranch_vccnz .LBB0_2', 's_nop 7', '.LBB0_2:\n', MFMA)[1]) == 1
    assert faults('s_branch .LBB0_2', '.LBB0_1:\n', 'v_mov_b32_e32 v9, v1', 's_endpgm', '.LBB0_2:\n', MFMA) == (1, [])
    # around two blocks of a loop
    assert len(faults(LOOP, MFMA, 's_cbranch_scc0 .LBB0_3', '.LBB0_2:\n', 'v_mov_b32_e32 v4, 0', AGAIN, '.LBB0_3:\n', 's_nop 0')[1]) == 1


def test_a_write_to_a_sum_that_is_not_there_yet_is_found():
    for write in ('v_accvgpr_write_b32 a2, 0', 'v_accvgpr_write_b32 a3, v1', 'ds_read_b128 a[0:3], v1', 'global_load_dword a1, v[2:3], off', 'v_accvgpr_mov_b32 a0, a9'):
        for between, bad in (([], 1), (['s_nop 15'], 1), (['s_nop 15', 's_nop 1'], 0)):
            assert len(faults(MFMA, *between, write)[1]) == bad, (write, between)


def test_a_product_that_takes_a_fresh_sum_is_found():
    own = '\t;;#ASMSTART\n\tv_mfma_f32_16x16x32_bf16 %s\n\t;;#ASMEND\n'
    for other in ('v_mfma_f32_16x16x32_bf16 a[8:11], a[0:3], v[8:11], a[8:11]', 'v_mfma_f32_16x16x32_bf16 a[8:11], v[8:11], a[2:5], a[8:11]',
                  'v_mfma_f32_16x16x32_bf16 a[8:11], v[4:7], v[8:11], a[0:3]', 'v_mfma_f32_16x16x32_bf16 a[2:5], v[4:7], v[8:11], a[2:5]',
                  'v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], 0'):
        assert len(faults(MFMA, other)[1]) == 1, other
        assert faults(MFMA, 's_nop 15', 's_nop 1', other) == (1, [])
        assert len(faults(MFMA, own % other.partition(' ')[2])[1]) == 1, other
    assert faults(MFMA, 'v_mfma_f32_16x16x32_bf16 a[0:3], v[12:15], v[16:19], a[0:3]') == (1, [])      # the sum goes on
    assert faults(own % 'v[0:3], v[4:7], v[8:11], 0', own % 'v[0:3], v[12:15], v[16:19], v[0:3]') == (2, [])
    assert len(faults(own % 'v[0:3], v[4:7], v[8:11], 0', 's_nop 3', 'v_add_f32_e32 v20, v20, v0')[1]) == 1


def test_every_way_of_storing_reads():
    for store in ('flat_store_dwordx4 v[20:21], a[0:3]', 'global_store_dword v[20:21], a0, off', 'global_atomic_add_f32 v20, a1, s[0:1]', 'global_atomic_pk_add_bf16 v[20:21], a3, off',
                  'buffer_atomic_add_f32 a2, off, s[0:3], 0', 'ds_add_f32 v20, a0', 'ds_write_b128 v20, a[0:3]', 'ds_write2_b32 v20, a0, a1 offset1:1', 'ds_bpermute_b32 v20, v21, a0',
                  'buffer_store_dwordx2 a[2:3], v20, s[0:3], 0 offen', 'flat_atomic_add v[20:21], a0', 'scratch_store_dword off, a1, s0'):
        assert len(faults(MFMA, store)[1]) == 1, store
        assert faults(MFMA, 's_nop 15', 's_nop 1', store) == (1, [])
    direct = '\t;;#ASMSTART\n\tbuffer_load_dwordx4 v9, s[0:3], s4 offen lds\n\t;;#ASMEND\n'      # straight to LDS: v9 is its address
    assert faults('v_mov_b32_e32 v9, v1', 's_nop 1', direct, MFMA) == (1, [])
    assert len(faults('v_mov_b32_e32 v9, v1', direct, MFMA)[1]) == 1


def test_scales_are_operands_too():
    scaled = '\t;;#ASMSTART\n\tv_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[8:15], v[16:23], a[0:3], v2, v3 op_sel_hi:[0,0,0]\n\t;;#ASMEND\n'
    for r in ('v2', 'v3', 'v15', 'v16'):
        assert len(faults('v_mov_b32_e32 %s, v1' % r, scaled)[1]) == 1
        assert faults('v_mov_b32_e32 %s, v1' % r, 's_nop 1', scaled) == (1, [])
