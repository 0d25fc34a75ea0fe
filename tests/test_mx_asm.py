"""The pipelined MXFP4 product (aiehlc_amd/csrc/gemm_mxfp4.hip, gemm_mx_pipe)
issues its matrix instructions through inline assembly, as the 16x16 int8 and
bf16 kernels do.  The same checks of the generated gfx950 assembly (this
build's, CPU only) as in test_gemm16_asm.py: no scratch memory, accumulators
updated in place, no instruction touches an accumulator before its result's
latency has passed, and no VALU instruction writes an operand or a scale within
three wait states before its use."""
import os
import subprocess

import pytest

import test_gemm16_asm as g

MFMA = "v_mfma_scale_f32_16x16x128_f8f6f4"


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not g._have_hipcc():
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asmmx") / "gemm_mxfp4.s"
    subprocess.run([g.HIPCC, *g.FLAGS, os.path.join(g.ROOT, "aiehlc_amd", "csrc", "gemm_mxfp4.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    return out.read_text()


@pytest.fixture()
def step(monkeypatch):
    """test_gemm16_asm's walk, which knows two sources and the accumulator, with the two scales as well."""
    plain = g._step

    def with_scales(name, t, state, mfma):
        if t.split()[0] == mfma:
            ops = [o.rstrip(",") for o in t.split()[1:]]
            scales = g._regs(ops[4]) | g._regs(ops[5])
            assert len(scales) in (1, 2) and "cbsz:4" in t and "blgp:4" in t, t
            for ago, regs in state[1]:
                assert not (regs & scales) or ago >= g.OPERAND_WAIT, f"{name}: scale written too soon before {t}"
        return plain(name, t, state, mfma)

    monkeypatch.setattr(g, "_step", with_scales)


def test_no_scratch(asm):
    g._check_no_scratch(asm, "gemm_mx_pipe")


def test_mfma_in_place_and_hazard_free(asm, step):
    assert g._check_hazards(asm, r"\S*gemm_mx_pipe\S*", MFMA) > 1000


def test_the_check_sees_a_scale_written_too_soon(step):
    text = ("f:\n\tv_lshrrev_b32 v9, 16, v9\n\ts_nop 0\n\tv_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:3], v[4:7], "
            "a[0:3], v8, v9 op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\ts_endpgm\n.Lfunc_end0:\n")
    with pytest.raises(AssertionError, match="scale written too soon"):
        g._check_hazards(text, "f", MFMA)
    assert g._check_hazards(text.replace("s_nop 0", "s_nop 2"), "f", MFMA) == 1
