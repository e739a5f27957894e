"""What must not be in the library's device code."""
from diffphycon_amd import _lib, build


def test_no_64_bit_shift_takes_its_amount_from_a_kernels_last_vector_register():
    """Where a wave's registers end the register file, such a shift was seen to take its amount from register 0."""
    assert build.last_register_shifts(build.device_asm(_lib.LIB_PATH)) == []


def test_the_scan_finds_such_a_shift():
    kernel = "0000000000001000 <%s>:\n\tv_mov_b32_e32 v%d, 0  // 000000001000: 7E000280\n\t%s  // 000000001004: 00000000\n"
    shift = "v_lshlrev_b64 v[4:5], v%d, 1"
    bad = kernel % ("bad", 14, shift % 15)
    assert build.last_register_shifts([bad]) == ["bad"]
    assert build.last_register_shifts([bad.replace("v_lshlrev_b64", "v_ashrrev_i64"), bad.replace("v_lshlrev_b64", "v_lshrrev_b64_e64")]) == ["bad", "bad"]
    fine = [kernel % ("below", 16, shift % 15), kernel % ("within", 12, shift % 13), kernel % ("constant", 15, "v_lshlrev_b64 v[4:5], 2, v[14:15]"),
            kernel % ("narrow", 14, "v_lshlrev_b32_e32 v4, v15, v4")]
    assert build.last_register_shifts(fine) == []
    assert build.last_register_shifts(["".join(fine) + bad]) == ["bad"]
