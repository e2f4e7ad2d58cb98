"""CPU tests of what the grouped products and the orthogonalised update say to operands that overlap: a result (or the workspace) on an
operand is refused, columns and rows beside one another are not taken for an overlap."""
import os
import subprocess

import pytest

from test_cpu_grouped_args import dw, gemm, ortho

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A, B, D, E, W = (1 << 20, 1 << 24, 1 << 28, 1 << 29, 1 << 30)   # addresses far from one another, never touched


def test_the_rule_against_sets_of_bytes(tmp_path):
    exe = str(tmp_path / "byte_rows_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-o", exe, os.path.join(ROOT, "tests", "cpp", "byte_rows_check.cpp")], check=True, timeout=300)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout


# rows of 16-bit elements: T = 4 of K = 8 and N = 6, two groups; the last element of one on the first of the other, the whole, columns
@pytest.mark.parametrize("over", [dict(Y=A), dict(Y=A + 62), dict(Y=B), dict(Y=B + 2 * 95), dict(Y=D), dict(Y=D + 22 - 24 * 2),
                                  dict(X=A, ldx=16, Y=A + 8, ldy=16), dict(X=A, ldx=16, Y=A + 22, ldy=16)], ids=str)
def test_grouped_gemm(over):
    assert gemm(**{**dict(X=A, W=B, off=D, Y=E), **over}) == 1


@pytest.mark.parametrize("over", [dict(c=A), dict(c=B + 46), dict(c=D), dict(c=W), dict(work=A), dict(work=E), dict(work=D), dict(c=A + 2 * 31)], ids=str)
def test_grouped_gemm_dw(over):
    # 2^20 rows of 64 in one group are cut into parts, which takes a workspace
    big = dict(dtype=1, cdtype=1, groups=1, T=1 << 20, M=64, N=64, ldx=64, ldz=64, ldc=64, sc=0, size=1 << 40)
    at = dict(X=1 << 32, Z=1 << 33, off=1 << 34, c=1 << 35, work=1 << 36)
    moved = {k: {A: at["X"], B + 46: at["Z"] + (1 << 26) + 4, D: at["off"], W: at["work"], E: at["c"], A + 2 * 31: at["X"] + (1 << 28) - 4}[v] for k, v in over.items()}
    assert dw(**{**big, **at, **moved}) == 1


@pytest.mark.parametrize("over", [dict(O=A + 4), dict(O=A, ldo=9, so=54), dict(O=A, so=52), dict(G=A, ldg=24, sg=192, O=A + 28, ldo=24, so=192),
                                  dict(work=A), dict(work=B + 64)], ids=str)
def test_orthogonalize(over):
    assert ortho(**{**dict(G=A, O=B, work=W), **over}) == 1
