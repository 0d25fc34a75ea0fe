"""The tiles of 8-bit products (aiehlc_amd/csrc/gemm_fp8.hip) issue their matrix
instructions through inline assembly, which the compiler's hazard recognizer does
not see.  These checks compile the file for gfx950 and read the assembly of this
build (CPU only):

- nothing is spilled, but for the two values that the mixed tiles of gate and up put
  away outside their loop;
- no instruction touches a product's registers before the product is there, 8 passes
  and 3 wait states after its issue, and no vector instruction writes an operand or a
  scale of a product within 3 wait states before it, along every branch.  A matrix
  instruction issues no sooner than 8 wait states behind the one before (measured:
  the instruction behind n of them issues 32 (n - 1) cycles after the first);
- a product that adds does so in place.
"""
import os
import re
import subprocess

import pytest

from test_gemm16_asm import FLAGS, HIPCC, ROOT, _functions, _have_hipcc, _is_branch, _items, _regs

PASSES, RESULT_WAIT, OPERAND_WAIT = 8, 8 + 3, 3
MFMA = re.compile(r"v_mfma_(scale_)?f32_16x16x128_f8f6f4 ")
PATTERN = r"_ZN5miaie\S*gemm_(?:tile|slots)\S*"


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not _have_hipcc():
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asmfp8") / "gemm_fp8.s"
    subprocess.run([HIPCC, *FLAGS, os.path.join(ROOT, "aiehlc_amd", "csrc", "gemm_fp8.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    return out.read_text()


def _state(results=(), writes=(), since=PASSES):
    """Products that are not there yet and late vector writes, each with its age, and the last product's age."""
    return list(results), list(writes), since


def _step(name, t, state):
    results, writes, since = state
    op = t.split()[0]
    ops = [o.rstrip(",") for o in t.split()[1:]]
    product = MFMA.match(t)
    if product:  # it waits for the one before
        wait = max(PASSES - since, 0)
        results = [(r, a + wait) for r, a in results if a + wait < RESULT_WAIT]
        writes = [(r, a + wait) for r, a in writes if a + wait < OPERAND_WAIT]
        since = 0
        dst, c = ops[0], ops[3]
        assert c == ("0" if not product.group(1) else dst), f"{name}: not in place: {t}"
        read = set().union(*(_regs(o) for o in ops[1:3] + ops[4:6]))
        for r, a in writes:
            assert not r & read, f"{name}: written {a} wait states before {t}"
        for r, a in results:
            assert not r & read, f"{name}: {t} reads a product after {a} wait states"
            assert not (r & _regs(dst)) or r == _regs(dst), f"{name}: {t} over a part of a product"
        results = [(r, a) for r, a in results if r != _regs(dst)] + [(_regs(dst), 0)]
    else:
        touched = set().union(*(_regs(o) for o in ops))
        for r, a in results:
            assert not r & touched, f"{name}: {t} touches a product after {a} wait states"
    step = int(ops[0]) + 1 if op == "s_nop" else 1
    results = [(r, a + step) for r, a in results if a + step < RESULT_WAIT]
    writes = [(r, a + step) for r, a in writes if a + step < OPERAND_WAIT]
    if op.startswith("v_") and not product and ops:
        writes.append((_regs(ops[0]), 0))
    return (results, writes, since + step), bool(product)


def _check(s, pattern):
    """Every kernel in text order; a branch carries its state to its target."""
    products = 0
    for name, body in _functions(s, pattern):
        items = _items(body)
        label_at = {t: i for i, (k, t) in enumerate(items) if k == "label"}
        incoming, back, state = {}, [], _state()
        for i, (kind, t) in enumerate(items):
            if kind == "label":
                for r, w, since in incoming.pop(t, []):
                    state = (state[0] + r, state[1] + w, max(state[2], since))
                continue
            state, n = _step(name, t, state)
            products += n
            if _is_branch(t.split()[0]):
                j = label_at[t.split()[1]]
                if j > i:
                    incoming.setdefault(items[j][1], []).append(state)
                else:
                    back.append((j, state))
                if t.split()[0] == "s_branch":
                    state = _state()  # nothing falls through
        for j, st in back:  # ... a loop's end to its head, until nothing of it is left
            for kind, t in items[j + 1:]:
                if not (st[0] or st[1]):
                    break
                if kind == "ins":
                    st, _ = _step(name, t, st)
                    # (what the head issues itself has been looked at above)
                    st = ([x for x in st[0] if not (x[1] <= 1 and MFMA.match(t))], [x for x in st[1] if x[1] > 0], st[2])
                    if _is_branch(t.split()[0]):
                        break
    return products


def test_products_keep_their_distances(asm):
    assert _check(asm, PATTERN) > 2000


def test_nothing_is_spilled(asm):
    meta, seen = asm[asm.index("amdhsa.kernels:"):], 0
    for blk in meta.split("\n  - ")[1:]:
        name = re.search(r"\.name:\s+(\S+)", blk)
        if not name:
            continue
        seen += 1
        scratch = int(re.search(r"\.private_segment_fixed_size:\s+(\d+)", blk).group(1))
        spilled = int(re.search(r"\.vgpr_spill_count:\s+(\d+)", blk).group(1))
        mixed_glu = "gemm_slots" in name.group(1) and "OutE2" in name.group(1)
        assert scratch <= 12 * mixed_glu and spilled <= 2 * mixed_glu, (name.group(1), scratch, spilled)
    assert seen >= 30


def _synthetic(*lines):
    return "f:\n" + "".join(f"\t{x}\n" if not x.endswith(":") else f"{x}\n" for x in lines) + "\ts_endpgm\n.Lfunc_end0:\n"


P0, P1, P2 = (f"v_mfma_f32_16x16x128_f8f6f4 v[{d}:{d + 3}], v[20:27], v[28:35], 0" for d in (0, 4, 8))
ACC = "v_mfma_scale_f32_16x16x128_f8f6f4 v[40:43], v[20:27], v[28:35], v[40:43], v50, v51 op_sel_hi:[0,0,0]"


def test_the_check_finds_what_it_is_for():
    add = "v_fmac_f32_e32 v60, v1, v61"
    assert _check(_synthetic(P0, P1, P2, add), "f") == 3
    with pytest.raises(AssertionError, match="touches a product"):
        _check(_synthetic(P0, P1, add), "f")
    assert _check(_synthetic(P0, P1, "s_nop 1", add), "f") == 2
    with pytest.raises(AssertionError, match="written"):
        _check(_synthetic("v_lshrrev_b32_e32 v50, 23, v52", "s_nop 1", ACC), "f")
    assert _check(_synthetic("v_lshrrev_b32_e32 v50, 23, v52", "s_nop 2", ACC), "f") == 1
    with pytest.raises(AssertionError, match="written"):  # around a loop
        _check(_synthetic(".LBB0_1:", ACC, "s_nop 7", "v_mov_b32_e32 v20, 0", "s_cbranch_scc1 .LBB0_1"), "f")
    with pytest.raises(AssertionError, match="touches a product"):
        _check(_synthetic(".LBB0_1:", add, P0, "s_cbranch_scc1 .LBB0_1"), "f")
    with pytest.raises(AssertionError, match="not in place"):
        _check(_synthetic(ACC.replace("v[40:43], v50", "v[44:47], v50")), "f")
    with pytest.raises(AssertionError, match="reads a product"):
        _check(_synthetic(P0, P1.replace("v[20:27]", "v[0:7]")), "f")
