"""tools/check_async_loads.py: an inline-asm load stands five wait states behind a vector instruction that writes one of its scalar
registers (the compiler's hazard recognizer does not look into inline asm)."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("check_async_loads", os.path.join(ROOT, "tools", "check_async_loads.py"))
chk = importlib.util.module_from_spec(spec)
spec.loader.exec_module(chk)


def run(between, tmp_path, writes="v_readlane_b32 s3, v126, 25"):
    p = tmp_path / "k.s"
    p.write_text(f"""_Z4kernPf:
\t{writes}
{between}\t;;#ASMSTART
\tglobal_load_dwordx4 v[10:13], v1, s[2:3]
\t;;#ASMEND
\ts_waitcnt vmcnt(0)
\ts_endpgm
\t.section\t.rodata
""")
    return chk.main([str(p)])


@pytest.mark.parametrize("writes", ["v_readlane_b32 s3, v126, 25", "v_readfirstlane_b32 s2, v7", "v_cmp_eq_u32_e64 s[2:3], 0, v7"])
def test_too_few_wait_states_fail(writes, tmp_path):
    for n in range(5):
        assert run("\tv_add_u32_e32 v5, v6, v7\n" * n, tmp_path, writes) == 1
    assert run("\tv_add_u32_e32 v5, v6, v7\n" * 5, tmp_path, writes) == 0
    assert run("\ts_nop 3\n", tmp_path, writes) == 1 and run("\ts_nop 4\n", tmp_path, writes) == 0


def test_other_registers_and_scalar_writes_pass(tmp_path):
    assert run("", tmp_path, "v_readlane_b32 s4, v126, 25") == 0
    assert run("\ts_addc_u32 s3, s7, s45\n", tmp_path) == 0
    assert run("\ts_mov_b32 s2, 0\n", tmp_path) == 1
