"""The build's dependencies: a changed header rebuilds every object whose source includes it, directly or through another header.  (An object left behind would
still link, and pass argument structs in an old layout.)"""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'edgegan_amd', 'csrc')
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(('.hip', '.cpp')))
HEADERS = sorted(f for f in os.listdir(CSRC) if f.endswith('.h')) + ['../../include/edgegan_hip.h']


def included(path, seen):
    """The project's headers that a file includes, as paths from CSRC."""
    with open(os.path.join(CSRC, path)) as f:
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', f.read(), re.M):
            p = os.path.normpath(os.path.join(os.path.dirname(path), name))
            if p not in seen and os.path.exists(os.path.join(CSRC, p)):
                seen.add(p)
                included(p, seen)
    return seen


@pytest.mark.parametrize('header', HEADERS + ['Makefile'])
def test_header_rebuilds_what_includes_it(header):
    if shutil.which('make') is None:
        pytest.skip('no make')
    out = subprocess.run(['make', '-n', '-W', header, '-C', CSRC], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr
    rebuilt = set(re.findall(r'-c (\S+) -o', out.stdout))
    users = SOURCES if header == 'Makefile' else [s for s in SOURCES if os.path.normpath(header) in included(s, set())]
    host = {'hostutil.cpp'} if header == 'Makefile' else set()      # (plain C++ with a rule of its own)
    missing = set(users) - rebuilt - host
    assert users and not missing, f'{header}: {sorted(missing)} would keep their old objects'
