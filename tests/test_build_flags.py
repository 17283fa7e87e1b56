"""CPU: the flags that results depend on reach every compilation, and a change to them compiles everything again."""
import os
import subprocess

import pytest

from helpers import ROOT

CSRC = os.path.join(ROOT, 'tempenslearnagg-qcnet_amd', 'csrc')
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith('.hip'))
REQUIRED = ('--offload-arch=gfx950', '-Xclang -target-feature -Xclang -packed-fp32-ops', '-mllvm -amdgpu-spill-vgpr-to-agpr=0', '-fPIC')


def _compilations(*args, **env):
    """What make would run (nothing is run), by source."""
    out = subprocess.run(['make', '-n', '-C', CSRC, *args], env=dict(os.environ, **env), check=True, capture_output=True, text=True).stdout
    lines = [' '.join(x.split()) for x in out.replace('\\\n', ' ').splitlines() if ' -c ' in x]
    return {f: x for f in SOURCES for x in lines if ' -c %s ' % f in x}


@pytest.mark.parametrize('args,env', [((), {}), ((), {'CXXFLAGS': '-O1'}), (('CXXFLAGS=-O1',), {})])
def test_required_flags_cannot_be_overridden(args, env):
    found = _compilations('-B', *args, **env)
    assert sorted(found) == SOURCES
    for line in found.values():
        assert all(flag in line for flag in REQUIRED), line
    assert '-fno-slp-vectorize' in found['fourier.hip']
    assert all('-O1' in x for x in found.values()) == bool(args or env)


def test_a_changed_makefile_compiles_everything_again():
    assert sorted(_compilations('-W', 'Makefile')) == SOURCES


def test_variants_take_the_same_flags():
    flags = subprocess.run(['make', '-s', '-C', CSRC, '--no-print-directory', 'flags'], check=True, capture_output=True, text=True).stdout
    assert all(flag in flags for flag in REQUIRED)
    for name in ('build_variant.sh', 'build_all_variant.sh'):
        with open(os.path.join(ROOT, 'scripts', 'dbg', name)) as f:
            assert '$(make -s flags)' in f.read()
