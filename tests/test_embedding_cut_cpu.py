"""Host-side checks of how an embedding gradient of few tokens is cut into launches
(csrc/embedding_cut.hpp): every row of the table once, each launch below 2^32 work-items."""
import os
import subprocess

from conftest import REPO

PROBE = r"""
#include <stdio.h>
#include "embedding_cut.hpp"
int main() {
    unsigned long long vocab, slabs;
    while (scanf("%llu %llu", &vocab, &slabs) == 2) {
        const ttp::FewRowsCut c = ttp::cut_few_rows(vocab, slabs, 256);
        printf("%u %llu\n", c.keys, (unsigned long long)c.rows);
    }
}
"""


def test_launches_of_few_tokens(tmp_path):
    (tmp_path / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    os.path.join(REPO, "tt-perf_amd", "csrc"), "-o", str(tmp_path / "probe"),
                    str(tmp_path / "probe.cpp")], check=True)
    tables = [(v, s) for v in (1, 2, 65, 4095, 50257, 2 ** 24 + 1, 2 ** 28 - 1, 2 ** 28, 2 ** 28 + 1,
                               2 ** 29 - 8, 2 ** 29, 2 ** 29 + 1003, 2 ** 30 - 1)
              for s in (1, 2, 3, 25, 1000, 2 ** 23) if v * s < 2 ** 34]
    out = subprocess.run([str(tmp_path / "probe")], input="".join("%d %d\n" % t for t in tables),
                         capture_output=True, text=True, check=True).stdout
    for (vocab, slabs), line in zip(tables, out.splitlines()):
        keys, rows = map(int, line.split())
        assert 1 <= keys <= 8 and rows % keys == 0 and rows > 0
        waves = -(-min(rows, vocab) // keys) * slabs
        assert -(-waves // 4) * 256 < 2 ** 32, (vocab, slabs)
        if vocab <= 2 ** 24 and slabs <= 25:  # one launch for a model's table
            assert rows >= vocab
    assert len(out.splitlines()) == len(tables)
