"""The build of the library: an object is as old as the flags it was compiled with, and a variant build keeps a source's own."""
import os
import stat
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def compiler(tmp_path):
    """A stand-in for hipcc that writes down its arguments, a call per line, and makes the file after -o."""
    log, exe = tmp_path / 'calls', tmp_path / 'hipcc'
    log.write_text('')
    exe.write_text('#!/bin/bash\necho "$@" >> %s\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then case "$2" in %s/*) touch "$2";; esac; fi; shift; done\n' % (log, tmp_path))
    exe.chmod(exe.stat().st_mode | stat.S_IEXEC)
    return str(exe), lambda: log.read_text().splitlines()


def test_a_change_of_flags_compiles_again(compiler, tmp_path, monkeypatch):
    from tacotron_amd import build as b
    exe, calls = compiler
    src = tmp_path / 'src'
    src.mkdir()
    for name in ('one.hip', 'two.hip', 'h.h'):
        (src / name).write_text('')
        os.utime(src / name, (1, 1))
    for name, x in dict(CSRC=str(src), OBJ=str(tmp_path / 'obj'), LIB=str(tmp_path / 'lib.so'), SOURCES=['one.hip', 'two.hip'],
                        HEADERS=['h.h'], HIPCC=exe, FLAGS=['-O3'], EXTRA_FLAGS={'two.hip': ['-x1']}).items():
        monkeypatch.setattr(b, name, x)
    b.build(verbose=False)
    assert len(calls()) == 3 and sum('-x1' in c for c in calls()) == 1
    b.build(verbose=False)
    assert len(calls()) == 3
    monkeypatch.setattr(b, 'EXTRA_FLAGS', {'two.hip': ['-x2']})
    b.build(verbose=False)
    assert len(calls()) == 5 and '-x2' in calls()[3] and 'two.hip' in calls()[3] and '-shared' in calls()[4]
    monkeypatch.setattr(b, 'FLAGS', ['-O2'])
    b.build(verbose=False)
    assert len(calls()) == 8
    b.build(verbose=False)
    assert len(calls()) == 8


@pytest.mark.parametrize('src,packed', [('kv_cache.hip', True), ('api.hip', False)])
def test_a_variant_build_keeps_the_flags_of_its_source(compiler, src, packed):
    from tacotron_amd import build as b
    exe, calls = compiler
    subprocess.run([os.path.join(ROOT, 'tools', 'build_any_variant.sh'), 'test', src, '-DWHAT=1'], check=True, env=dict(os.environ, HIPCC=exe),
                   capture_output=True)
    compiled, linked = calls()
    assert all(f in compiled.split() for f in b.FLAGS + ['-DWHAT=1', '-c', 'tacotron_amd/csrc/' + src])
    assert ('-packed-fp32-ops' in compiled) == packed
    assert all(('/%s%s.o' % (s[:-4], '_test' if s == src else '')) in linked for s in b.SOURCES)


def test_the_build_entry_compiles_whatever_is_there(monkeypatch):
    """It is the check that the sources build, so an object from before is no reason to leave one out."""
    import __graft_entry__ as g
    from tacotron_amd import build as b
    asked = []
    monkeypatch.setattr(b, 'build', lambda force=False, verbose=True: asked.append(force) or b.LIB)
    g.build()
    assert asked == [True]
