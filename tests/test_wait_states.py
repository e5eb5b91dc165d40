"""The compiler's listing of shared_prefix.hip: no instruction touches what a matrix product
writes before the product is through. The hardware does not wait there, the compiler counts
instructions; where two paths meet right behind products, one of them without instructions,
it has been seen to leave its count out."""

import ast
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "parallax_amd", "ops", "csrc")
# wait states from a product of this shape to the next use of its result on gfx950: its
# passes of four cycles, and four
STATES = {"16x16x32": 4 + 4, "32x32x16": 8 + 4}


def _flags():
    """HIP_FLAGS of setup.py."""
    with open(os.path.join(ROOT, "setup.py")) as f:
        tree = ast.parse(f.read())
    names = {}
    for node in tree.body:
        if isinstance(node, ast.Assign) and node.targets[0].id == "HIP_FLAGS":
            exec(compile(ast.Module([node], []), "setup.py", "exec"), names)
    return names["HIP_FLAGS"]


def _registers(operand):
    return {int(r) for a, b, one in re.findall(
        r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", operand)
        for r in (range(int(a), int(b) + 1) if a else (one,))}


def _functions(listing):
    """name -> (instructions as (name, operands), label -> place) of every kernel."""
    found = {}
    for name, body in re.findall(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end", listing,
                                 re.S | re.M):
        code, labels = [], {}
        for line in body.split("\n"):
            line = line.split(";")[0].rstrip()
            label = re.match(r"(\.LBB\w+):", line)
            if label:
                labels[label.group(1)] = len(code)
            elif line.startswith("\t") and line.strip() and line.strip()[0] != ".":
                op, _, rest = line.strip().partition(" ")
                code.append((op, rest.split(", ") if rest else []))
        found[name] = code, labels
    return found


def _too_early(code, labels):
    """(product, instruction, wait states between them) of all that are too close."""
    bad = []
    for at, (op, args) in enumerate(code):
        if "mfma" not in op:
            continue
        need = next(n for shape, n in STATES.items() if shape in op)
        result = _registers(args[0])
        paths, least = [(at + 1, 0)], {}
        while paths:
            i, states = paths.pop()
            if i >= len(code) or states >= need or least.get(i, need) <= states:
                continue
            least[i] = states
            name, given = code[i]
            if "mfma" in name:
                # the accumulators of the next product are handed on without a wait
                if (_registers(given[1]) | _registers(given[2])) & result:
                    bad.append((at, i, states))
                if _registers(given[0]) & result:
                    continue
            elif not name.startswith("s_"):
                if any(_registers(x) & result for x in given):
                    bad.append((at, i, states))
                    continue
            if name == "s_endpgm":
                continue
            then = states + 1 + (int(given[0], 0) if name == "s_nop" else 0)
            if name.startswith(("s_branch", "s_cbranch")):
                paths.append((labels[given[0]], then))
            if name != "s_branch":
                paths.append((i + 1, then))
    return bad


def test_the_check_sees_them():
    """A value read at once, one read behind its wait, one read early on one path only."""
    text = """_Zk:
\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]
{}
\ts_endpgm
.Lfunc_end0:
"""
    def early(lines):
        (code, labels), = _functions(text.format(lines)).values()
        return len(_too_early(code, labels))

    assert early("\tv_add_f32_e32 v4, v3, v5") == 1
    assert early("\ts_nop 6\n\tv_add_f32_e32 v4, v3, v5") == 1
    assert early("\ts_nop 7\n\tv_add_f32_e32 v4, v3, v5") == 0
    assert early("\tds_write_b32 v20, v2") == 1
    assert early("\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]") == 0
    assert early("\tv_mfma_f32_16x16x32_bf16 v[4:7], v[0:3], v[12:15], v[4:7]") == 1
    assert early("\ts_cbranch_scc0 .LBB0_1\n\ts_nop 7\n.LBB0_1:\n"
                 "\tv_add_f32_e32 v4, v3, v5") == 1


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")
def test_products_are_waited_for(tmp_path):
    out = tmp_path / "listing.s"
    subprocess.run(
        ["hipcc", *_flags(), "--offload-arch=gfx950", "--cuda-device-only", "-S",
         os.path.join(CSRC, "shared_prefix.hip"), "-o", str(out)], check=True,
        capture_output=True)
    kernels = _functions(out.read_text())
    assert sum(any("mfma" in op for op, _ in code)
               for code, _ in kernels.values()) == 8
    for name, (code, labels) in kernels.items():
        early = [(*map(lambda i: " ".join([code[i][0], ", ".join(code[i][1])]), (a, b)), n)
                 for a, b, n in _too_early(code, labels)]
        assert not early, (name, early[:5])
