"""CPU: the build's lists name every header that a translation unit includes, directly or through others, so
that a change to a header rebuilds each object that holds its code."""
import os
import re

import pytest

from muxi_race_b200 import build


def included(path, seen):
    for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', open(path).read(), re.M):
        full = os.path.normpath(os.path.join(os.path.dirname(path), name))
        if full not in seen:
            seen.add(full)
            included(full, seen)
    return seen


@pytest.mark.parametrize("source", sorted(build.SOURCES))
def test_headers_of(source):
    named = {os.path.normpath(os.path.join(build.CSRC, h)) for h in build.SOURCES[source] + build.API_HEADERS}
    assert included(os.path.join(build.CSRC, source), set()) <= named


def test_every_source_is_listed():
    assert set(build.SOURCES) == {f for f in os.listdir(build.CSRC) if f.endswith(".cu")}
