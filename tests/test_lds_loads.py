"""tools/check_lds_loads.py: the static check that nothing but the loads to LDS touches m0 in a compiled kernel."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("check_lds_loads", os.path.join(ROOT, "tools", "check_lds_loads.py"))
chk = importlib.util.module_from_spec(spec)
spec.loader.exec_module(chk)

GOOD = """
\t;;#ASMSTART
\ts_mov_b32 m0, s7
\ts_nop 3
\tbuffer_load_dwordx4 v3, s[8:11], 0 offen lds
\t;;#ASMEND
\tv_add_f32_e32 v2, v3, v4   ; m0 in a comment
\tbuffer_load_dwordx4 v[4:7], v3, s[8:11], 0 offen
"""


def run(body, tmp_path):
    p = tmp_path / "k.s"
    p.write_text(body)
    return chk.main([str(p)])


def test_a_move_and_its_load_pass(tmp_path):
    assert run(GOOD, tmp_path) == 0


@pytest.mark.parametrize("line", ["\ts_mov_b32 m0, s3\n", "\tv_movrels_b32_e32 v1, m0\n", "\tbuffer_load_dword v3, s[8:11], 0 offen lds\n",
                                  "\t;;#ASMSTART\n\ts_nop 0\n\tbuffer_load_dword v3, s[8:11], 0 offen lds\n\t;;#ASMEND\n"])
def test_other_uses_of_m0_and_loads_without_a_move_fail(line, tmp_path):
    assert run(GOOD + line, tmp_path) == 1


def test_a_load_too_close_behind_a_scalar_register_fails(tmp_path):
    for nop in range(3):
        assert run(GOOD.replace("s_nop 3", f"s_nop {nop}"), tmp_path) == 1


def test_a_listing_without_such_loads_fails(tmp_path):
    assert run("\ts_endpgm\n", tmp_path) == 1
