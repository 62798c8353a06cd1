"""CPU: the layout of include/b200seq.h's structs, as a C compiler sees it, as ctypes mirrors it and as the version says it."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from blazr_b200 import seqops

HEADER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include", "b200seq.h")
# bytes of every struct in each version: a struct that changes makes a new version and gets a line of its own here
SIZES = {2: dict(b200seq_step=64, b200seq_attn_desc=208, b200seq_retention_desc=96, b200seq_route_desc=40, b200seq_delta_desc=88, b200seq_scan_desc=48, b200seq_parallel_desc=176)}
MIRRORS = dict(b200seq_step=seqops.StepDesc, b200seq_attn_desc=seqops.AttnDesc, b200seq_retention_desc=seqops.RetentionDesc, b200seq_route_desc=seqops.RouteDesc,
               b200seq_delta_desc=seqops.DeltaDesc, b200seq_scan_desc=seqops.ScanDesc, b200seq_parallel_desc=seqops.ParallelDesc)


def test_every_struct_has_a_mirror():
    assert set(re.findall(r"^typedef struct (\w+)", open(HEADER).read(), re.M)) == set(MIRRORS)


def test_structs_are_those_of_the_version(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = {n: [f[0] for f in m._fields_] for n, m in MIRRORS.items()}
    src = ['#include <stddef.h>', '#include <stdio.h>', f'#include "{os.path.abspath(HEADER)}"', "int main(void) {", 'printf("%d\\n", B200SEQ_VERSION);']
    for n, fs in fields.items():
        src.append(f'printf("{n} %zu' + " %zu" * len(fs) + f'\\n", sizeof({n}), ' + ", ".join(f"offsetof({n}, {f})" for f in fs) + ");")
    (tmp_path / "a.c").write_text("\n".join(src + ["return 0;", "}"]))
    subprocess.run([cc, "-o", str(tmp_path / "a"), str(tmp_path / "a.c")], check=True)
    version, *rest = subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {r.split()[0]: [int(x) for x in r.split()[1:]] for r in rest if r}
    for n, m in MIRRORS.items():
        assert got[n] == [C.sizeof(m)] + [getattr(m, f).offset for f in fields[n]], n
    assert {n: v[0] for n, v in got.items()} == SIZES[int(version)]


def test_the_library_is_of_the_header_s_version():
    version = int(re.search(r"#define B200SEQ_VERSION (\d+)", open(HEADER).read()).group(1))
    assert seqops.lib().b200seq_version() == version == seqops.VERSION
