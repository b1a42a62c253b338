"""tools/check_spills.py: no register is put away at a join before the lanes that were off are on again."""
import glob
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("check_spills", os.path.join(ROOT, "tools", "check_spills.py"))
chk = importlib.util.module_from_spec(spec)
spec.loader.exec_module(chk)


def run(block, tmp_path):
    p = tmp_path / "k.s"
    p.write_text("_Z4kernPf:\n\ts_cbranch_execz .LBB0_2\n\tglobal_load_dword v5, v[0:1], off\n.LBB0_2:\n" + block + "\ts_endpgm\n")
    return chk.main([str(p)])


def test_a_spill_behind_the_join_passes(tmp_path):
    assert run("\ts_or_b64 exec, exec, s[2:3]\n\tv_accvgpr_write_b32 a2, v66\n", tmp_path) == 0
    assert run("\tv_accvgpr_write_b32 a1, 0\n\tv_mov_b32_e32 v4, v5\n\ts_or_b64 exec, exec, s[2:3]\n", tmp_path) == 0
    assert run("\tv_accvgpr_write_b32 a2, v66\n\ts_branch .LBB0_3\n", tmp_path) == 0


@pytest.mark.parametrize("spill", ["v_accvgpr_write_b32 a2, v66", "scratch_store_dword off, v66, off", "buffer_store_dword v66, off, s[0:3], 0"])
def test_a_spill_in_front_of_it_fails(spill, tmp_path):
    assert run(f"\tv_mov_b32_e32 v4, v5\n\t{spill}\n\ts_or_b64 exec, exec, s[2:3]\n", tmp_path) == 1


def test_the_built_kernels_pass():
    files = sorted(glob.glob(os.path.join(ROOT, "tsdiff_amd", "csrc", "*.verify.s")))
    if not files:
        pytest.skip("no kernel listings (run `make -C tsdiff_amd/csrc`)")
    assert chk.main(files) == 0
