"""CPU: which batches get a pass of their own for their prefixes (csrc/latent_plan.hpp), and that the tables with which
the GPU tests ask for one do get it."""
import os
import shutil
import subprocess
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    """[(G, B, T, H, keys)] -> the rule's answers."""
    at = tmp_path_factory.mktemp("rule")
    (at / "rule.cpp").write_text(
        '#include <cstdio>\n#include "latent_plan.hpp"\nint main() { int g, b, t, h; long long k; while (std::scanf('
        '"%d %d %d %d %lld", &g, &b, &t, &h, &k) == 5) std::puts(ferret::latent_prefix_pass(g, b, t, h, k) ? "1" : "0"); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{ROOT}/ferret_amd/csrc", str(at / "rule.cpp"), "-o",
                    str(at / "rule")], check=True)

    def ask(rows):
        out = subprocess.run([str(at / "rule")], input="\n".join("%d %d %d %d %d" % r for r in rows), capture_output=True,
                             text=True, check=True).stdout
        return [x == "1" for x in out.split()]
    return ask


def test_partials_of_many_rows_are_counted(rule):
    """The keys from which a pass pays grow with the rows: 512 sequences of 32 heads behind one prefix took 105 us in two
    passes and 86 in one at 512 keys, 148 and 160 at 2048."""
    assert rule([(1, 512, 512, 32, 512), (1, 512, 512, 32, 2048), (1, 400, 400, 32, 512), (1, 400, 400, 16, 1024)]) == [
        False, True, False, True]
    for H in (8, 16, 32):
        pays = []
        for B in (64, 128, 256, 512, 1024, 4096):
            answers = rule([(1, B, B, H, 64 * k) for k in range(1, 4000)])
            assert answers == sorted(answers), "more keys, no pass again"
            pays.append((answers.index(True) + 1) * B)      # steps of all sequences
        assert pays[-1] > pays[0], (H, pays)


def test_few_rows_as_before(rule):
    """Up to 6400 rows the steps alone decide."""
    got = rule([(1, 64, 64, 16, 8192), (1, 64, 64, 16, 2000), (8, 64, 64, 16, 2624), (1, 16, 16, 16, 8192),
                (1, 32, 32, 128, 1 << 20), (1, 4, 4, 16, 512), (21, 63, 63, 16, 6000), (1, 1, 1, 16, 1 << 30)])
    assert got == [True, False, True, False, False, False, False, False]


def test_the_tables_of_the_gpu_tests(rule, monkeypatch):
    """Shared.wide() says whether rows allow a pass, and makes a table that is wide enough for one."""
    from tests.test_gpu_shared_attention import Shared
    full = torch.full
    monkeypatch.setattr(torch, "full", lambda *a, **kw: full(*a, **{k: v for k, v in kw.items() if k != "device"}))
    asked, wanted = [], []
    for H in (1, 4, 5, 8, 16, 17, 24, 32, 64):
        for G in (1, 2, 3, 7):
            for members in (1, 2, 4, 7, 9, 30, 60):
                for new in (1, 2):
                    s = object.__new__(Shared)
                    s.H, s.G, s.page, B = H, G, 16, G * members
                    s.own, s.new = [(1, new)] * B, [new] * B
                    s.index = types.MethodType(lambda self: {"prefix_table": torch.zeros((self.G, 1), dtype=torch.int32)}, s)
                    if B * new * H > 6400:
                        continue
                    kw = s.wide()
                    keys = 1 << 30 if kw is None else kw["prefix_table"].shape[1] * s.page
                    asked.append((G, B, B * new, H, keys))
                    wanted.append(kw is not None)
    assert rule(asked) == wanted and 50 < sum(wanted) < len(wanted) - 50
