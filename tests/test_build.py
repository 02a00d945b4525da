"""The build's list of what the library is made of."""
import importlib.util
import os
import re

from conftest import ROOT


def test_a_change_to_any_included_file_rebuilds_the_library():
    spec = importlib.util.spec_from_file_location("b200attn_build", os.path.join(ROOT, "accelerated-final-project_b200", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    known = {os.path.realpath(p) for p in build.deps()}
    for path in sorted(known):
        for name in re.findall(r'#include "([^"]+)"', open(path).read()):
            at = os.path.realpath(os.path.join(os.path.dirname(path), name))
            assert at in known, (path, name)
