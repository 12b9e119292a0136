"""CPU: the build's look at inline matrix instructions, on assembly written here."""
import importlib.util
import os

from conftest import PKG

_at = os.path.join(PKG, "csrc", "check_pinned.py")
_spec = importlib.util.spec_from_file_location("check_pinned", _at)
check_pinned = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(check_pinned)

_MFMA = """	;;#ASMSTART
	v_mfma_f32_16x16x32_bf16 a[0:3], v[{a}:{a3}], v[8:11], a[0:3]
	;;#ASMEND
"""


def _mfma(a=4):
    return _MFMA.format(a=a, a3=a + 3)


def _kernel(before="", first="", between="", tail="", behind="	s_nop 15\n	s_nop 15\n"):
    return f"""kernel:                                 ; @kernel
	v_accvgpr_write_b32 a0, 0
	s_nop 7
{before}.LBB0_1:                                ; =>This Inner Loop
	ds_read_b128 v[4:7], v20
	s_waitcnt lgkmcnt(0)
{first}{_mfma()}{between}{_mfma(12)}{tail}	s_cbranch_scc1 .LBB0_1
{behind}	v_accvgpr_read_b32 v1, a0
	s_endpgm
other:
	v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]
	s_endpgm
"""


def _wrong(**parts):
    found = {name: check_pinned.check(body)
             for name, body in check_pinned.kernels(_kernel(**parts)).items()}
    assert found["other"] is None
    return found["kernel"]


def test_clean_assembly_passes(tmp_path):
    assert _wrong() == []
    assert _wrong(between="	v_add_u32 v30, v31, v32\n	ds_read_b128 v[16:19], v20\n") == []
    assert _wrong(between="	v_add_u32 v12, v31, v32\n	s_nop 3\n") == []
    assert _wrong(tail="	v_add_u32 v8, v31, v32\n	s_nop 1\n	s_nop 0\n") == []
    path = tmp_path / "unit.s"
    path.write_text(_kernel())
    assert check_pinned.main(str(path), 1) == 0
    assert check_pinned.main(str(path), 2) == 1


def test_moves_of_the_sums_are_found(tmp_path):
    for move in ("	v_accvgpr_read_b32 v9, a2\n", "	v_accvgpr_mov_b32 a9, a1\n",
                 "	ds_write_b128 v9, a[0:3]\n"):
        assert any("touches the sums" in w for w in _wrong(between=move)), move
    path = tmp_path / "unit.s"
    path.write_text(_kernel(between="	v_accvgpr_read_b32 v9, a2\n"))
    assert check_pinned.main(str(path), 1) == 1


def test_operands_written_too_late_are_found():
    for parts in (dict(first="	v_mov_b32_e32 v5, v40\n"), dict(first="	v_mov_b32_e32 v11, v40\n	s_nop 1\n"),
                  dict(between="	v_pk_mul_f16 v15, v1, v2\n	s_nop 2\n"),
                  dict(tail="	v_mov_b32_e32 v9, v1\n"),  # through the loop's end
                  dict(before="	v_mov_b32_e32 v10, v1\n	s_nop 0\n"),
                  dict(before="	v_accvgpr_write_b32 a3, 0\n")):
        assert any("right before" in w for w in _wrong(**parts)), parts


def test_sums_read_too_early_are_found():
    # 19 wait states, of which the loop's branch is one
    for wait in ("", "	s_nop 15\n", "	s_nop 15\n	s_nop 0\n"):
        assert any("behind the last" in w for w in _wrong(behind=wait)), wait
    assert _wrong(behind="	s_nop 15\n	s_nop 1\n") == []
