"""CPU: build() with a compiler that only notes how it was called."""
import os
import stat

import pytest

import __graft_entry__ as entry


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    from oracle_amd import _lib
    log, tools, csrc = tmp_path / 'log', tmp_path / 'bin', tmp_path / 'csrc'
    tools.mkdir(), csrc.mkdir()
    hipcc = tools / 'hipcc'
    hipcc.write_text(f'#!/bin/bash\n[ "$1" = --version ] && exit 0\necho "$@" >> {log}\n[ -e {tmp_path}/broken ] && exit 1\n'
                     'while [ "$1" != -o ]; do shift; done; echo "$RANDOM" > "$2"\n')
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv('PATH', f'{tools}:{os.environ["PATH"]}')
    monkeypatch.setattr(entry, 'CSRC', str(csrc))
    monkeypatch.setattr(_lib, 'lib', lambda: None)
    for name in entry.SOURCES + ['common.h', 'kernels.h', 'mma16.h', 'flash32.h']:
        (csrc / name).write_text('')
    return tmp_path, lambda: log.read_text().split('\n')[:-1] if log.exists() else []


def test_every_build_compiles_every_source(compiler):
    root, calls = compiler
    lib = root / 'csrc' / 'liboracle_hip.so'
    for i in range(1, 4):
        entry.build()
        assert lib.exists() and len(calls()) == i * (len(entry.SOURCES) + 1)
        new = calls()[-len(entry.SOURCES) - 1:]
        assert all(sum(c.endswith('/' + s) and '--offload-arch=gfx950' in c and '-packed-fp32-ops' in c for c in new) == 1 for s in entry.SOURCES)


def test_a_library_in_use_is_replaced_not_written_over(compiler):
    root, _ = compiler
    lib = root / 'csrc' / 'liboracle_hip.so'
    entry.build()
    with open(lib) as f:
        old = f.read()
        entry.build()
        f.seek(0)
        assert f.read() == old and lib.stat().st_ino != os.fstat(f.fileno()).st_ino
    (root / 'broken').write_text('')
    kept = lib.read_bytes()
    with pytest.raises(RuntimeError, match='hipcc failed'):
        entry.build()
    assert lib.read_bytes() == kept and sorted(p.name for p in (root / 'csrc').iterdir() if p.suffix not in ('.hip', '.h')) == ['liboracle_hip.so']
