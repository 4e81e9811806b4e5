"""The rules that choose a kernel's form (csrc/mx_rule.h), on the CPU: the GPU tests' shapes take the forms that they
are there for, and those are all the forms there are."""
import os
import random
import shutil
import subprocess

import pytest

import expert_forms as F
from tinyoai_amd import weights as W

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host compiler")
    exe = str(tmp_path_factory.mktemp("rule") / "rule_test")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "tinyoai_amd", "csrc"),
                    os.path.join(ROOT, "tests", "rule_test.cpp"), "-o", exe], check=True)

    def ask(lines):
        r = subprocess.run([exe], input="\n".join(lines), capture_output=True, text=True)
        assert r.returncode == 0, r.returncode
        out = [tuple(int(v) if v.isdigit() else v for v in line.split()) for line in r.stdout.splitlines()]
        assert len(out) == len(lines)
        return out

    return ask


def _line(fmt, xd, gate, grouped, experts, n, rows, cols):
    return f"p {int(fmt == W.BF16)} {F.PLANES[xd]} {int(gate)} {int(grouped)} {experts} {n} {rows} {cols}"


def test_every_product_form(rule):
    cases = [*F.few_forms(), *F.tile_forms()]
    got = rule([_line(c.fmt, c.xdtype, c.gate, True, len(c.counts), sum(c.counts) + F.TAIL, c.rows, c.cols) for c in cases])
    for c, g in zip(cases, got):
        assert g == c.form, c
    runs = [*F.run_forms()]
    got = rule([_line(fmt, xd, False, True, 1, n, rows, cols) for _, fmt, xd, n, rows, cols in runs])
    for c, g in zip(runs, got):
        assert g == c[0], c
    # of each pair of types: what csrc/mx_few.hip and csrc/mx_tiles.hip make of the rules' answers
    seen = {(c.fmt, c.xdtype, c.gate, *c.form) for c in cases} | {(c[1], c[2], False, *c[0]) for c in runs}
    for fmt, xd in F.PAIRS:
        for gate in (False, True):
            few = [("few", 8, t, k) for t in (1, 2) for k in (3, 4)] + [("few", 16, 1, 4)] * (not gate or xd == W.MXFP4)
            large = [(256, 256)] * (fmt == W.BF16 and xd == W.BF16) + [(128, 256)] * (fmt == W.BF16 or xd == W.MXFP4)
            tiles = [("tile", *t, 0) for t in [(32, 128), (64, 128), (64, 256), *large]]
            want = few + tiles
            if not gate:
                want += [("tile", *t, 1) for t in [(32, 128), (64, 128), (64, 256)] + [(128, 256)] * (fmt == W.BF16)]
            assert {s[3:] for s in seen if s[:3] == (fmt, xd, gate)} == set(want), (fmt, xd, gate)


def test_rules_of_any_sizes(rule):
    """No answer but those forms, and products in parts on the smallest tiles alone (the filter's exit code)."""
    rng = random.Random(1)
    lines, cases = [], []
    for _ in range(20000):
        fmt, xd = rng.choice(F.PAIRS)
        log = lambda hi: int(2 ** rng.uniform(0, hi))  # noqa: E731
        gate, grouped = rng.random() < 0.5, rng.random() < 0.6
        cases.append((fmt, xd))
        lines.append(_line(fmt, xd, gate and grouped, grouped, log(16) if grouped else 1, log(22), log(16), 32 * log(17)))
    for (fmt, xd), g in zip(cases, rule(lines)):
        if g[0] == "few":
            assert g[1:] in ((8, 1, 3), (8, 2, 3), (8, 1, 4), (8, 2, 4), (16, 1, 4))
        else:
            allowed = [(32, 128, 0), (32, 128, 1), (64, 128, 0), (64, 128, 1), (64, 256, 0), (64, 256, 1)]
            allowed += [(128, 256, 0)] * (fmt == W.BF16 or xd == W.MXFP4) + [(128, 256, 1)] * (fmt == W.BF16)
            allowed += [(256, 256, 0)] * (fmt == W.BF16 and xd == W.BF16)
            assert g[1:] in allowed


def test_every_routing_form(rule):
    got = rule([f"r {n} {experts} {k}" for _, n, experts, k in F.ROUTES])
    assert got == [form for form, *_ in F.ROUTES]
    assert {form for form, *_ in F.ROUTES} == {(p, e) for p in ("one_block", "by_expert", "by_tokens") for e in (1, 2, 4, 8, 16)}


def test_many_experts_leave_the_streaming_kernel(rule):
    """32 experts and more of large matrices at half of the rows: their groups may be uneven."""
    def form(experts, n, rows=1728, cols=2560, xd=W.BF16):
        return rule([_line(W.MXFP4, xd, True, True, experts, n, rows, cols)])[0][0]

    assert [form(64, 16 * 64), form(64, 16 * 64 + 1), form(64, 32 * 64)] == ["few", "tile", "tile"]
    assert [form(64, 16 * 64 // 3, xd=W.F32), form(64, 16 * 64 // 3 + 1, xd=W.F32)] == ["few", "tile"]
    assert [form(8, 32 * 8), form(8, 32 * 8 + 1)] == ["few", "tile"]
    assert [form(32, 32 * 32, 256, 1024), form(32, 32 * 32 + 1, 256, 1024)] == ["few", "tile"]
