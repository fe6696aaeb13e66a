"""The build-time scan for readers right behind an exponential or its like (int_flashattention_amd/mfma_check.py) on hand-made assembly."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "int-flashattention_amd"))
import mfma_check  # noqa: E402

HEAD = "_ZN5intfa4kernEv:\n\ts_load_dwordx2 s[0:1], s[4:5], 0x0\n"
TAIL = "\ts_endpgm\n"


@pytest.mark.parametrize("op", ["v_exp_f32_e32", "v_log_f32_e32", "v_rcp_f32_e32", "v_sqrt_f32_e32", "v_rsq_f32_e32", "v_rcp_iflag_f32_e32", "v_sin_f32_e32"])
@pytest.mark.parametrize("reader", ["v_fmac_f32_dpp v7, v8, v4 row_newbcast:3 row_mask:0xf bank_mask:0xf", "v_mul_f32_e32 v5, v4, v6", "v_fmac_f32_e32 v4, v5, v6",
                                    "v_cvt_pk_f16_f32 v5, v3, v4", "v_pk_add_f16 v5, v[4:5], v6"])
def test_a_reader_needs_one_state(op, reader):
    trans, read = f"\t{op} v4, v9\n", f"\t{reader} ; v4\n"
    found = mfma_check.scan_trans(HEAD + trans + read + TAIL)
    assert len(found) == 1 and "line 4" in found[0] and "of line 3" in found[0]
    for between in ("\ts_nop 0\n", "\tv_mov_b32_e32 v60, 0\n", "\ts_mov_b32 s3, 0\n"):
        assert mfma_check.scan_trans(HEAD + trans + between + read + TAIL) == []


def test_what_needs_none():
    trans = HEAD + "\tv_exp_f32_e32 v4, v9\n"
    for line in ("v_exp_f32_e32 v5, v4", "v_mov_b32_e32 v4, v5", "v_add_f32_e32 v5, v6, v14", "ds_write_b32 v7, v4", "v_mul_f32_e32 v5, s4, v6"):
        assert mfma_check.scan_trans(trans + "\t" + line + "\n" + TAIL) == []
    # an empty hand-written statement is no wait state
    assert len(mfma_check.scan_trans(trans + "\t;;#ASMSTART\n\t;;#ASMEND\n\tv_add_f32_e32 v5, v4, v6\n" + TAIL)) == 1


def test_every_way_on_is_followed():
    asm = HEAD + "\tv_mov_b32_e32 v1, 0\n\tv_exp_f32_e32 v4, v9\n.LBB0_1:\n{}\tv_add_f32_e32 v5, v4, v6\n" + TAIL
    assert len(mfma_check.scan_trans(asm.format(""))) == 1
    assert mfma_check.scan_trans(asm.format("\ts_nop 0\n")) == []
    # a branch is a state of its own
    assert mfma_check.scan_trans(HEAD + "\tv_exp_f32_e32 v4, v9\n\ts_cbranch_scc1 .LBB0_1\n; %bb.1:\n\tv_add_f32_e32 v5, v4, v6\n.LBB0_1:\n\tv_add_f32_e32 v5, v4, v6\n" + TAIL) == []
