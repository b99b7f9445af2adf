"""The Makefile names for every object the headers that its source takes, so that none is left of before an edit."""

import pathlib
import re
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "distdl_amd" / "csrc"
SOURCES = sorted(p.name for p in CSRC.iterdir() if p.suffix in (".hip", ".cpp"))


def headers_of(path, seen=()):
    """All that ``path`` includes of this repository, as seen from csrc."""
    found = set()
    for name in re.findall(r'#include "([^"]+)"', path.read_text()):
        header = (path.parent / name).resolve()
        if header not in found and header not in seen:
            found |= {header} | headers_of(header, found | set(seen))
    return found


@pytest.mark.parametrize("source", SOURCES)
def test_an_edited_header_compiles_what_includes_it(source):
    target = "../libdistdl_bench_probes.so" if source.startswith("bench_probes") else "build/" + source.rsplit(".", 1)[0] + ".o"
    for header in sorted(headers_of(CSRC / source)) + [CSRC / source]:
        name = str(header.relative_to(CSRC)) if header.parent == CSRC else "../../include/" + header.name
        plan = subprocess.run(["make", "-C", str(CSRC), "-n", "-W", name, target], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, check=True).stdout
        assert re.search(r"-o \S*" + re.escape(target), plan), f"{target} stays as it is when {name} changes"
