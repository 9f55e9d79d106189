"""asr_amd.build: what is compiled again, with a stand-in for the compiler."""
import os
import stat

import pytest

from asr_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of two sources, a header and a recipe, all older than anything made from them, and a compiler that writes its output file and its command down."""
    csrc = tmp_path / 'asr_amd' / 'csrc'
    csrc.mkdir(parents=True)
    for name in ('a.hip', 'b.hip', 'x.h', 'recipe.py'):
        (csrc / name).write_text(name)
        os.utime(csrc / name, (1000, 1000))
    log = tmp_path / 'log'
    log.write_text('')
    hipcc = tmp_path / 'hipcc'
    hipcc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ "$1" != -o ]; do shift; done\necho made > "$2"\n' % log)
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv('HIPCC', str(hipcc))
    for name, value in (('CSRC', str(csrc)), ('LIB', str(csrc / 'lib.so')), ('SOURCES', ['a.hip', 'b.hip']), ('HEADERS', ['x.h']),
                        ('RECIPE', str(csrc / 'recipe.py'))):
        monkeypatch.setattr(build, name, value, raising=name != 'RECIPE')

    def made(force=False):
        log.write_text('')
        build.build_library(force=force, verbose=False)
        lines = log.read_text().splitlines()
        for name in ('a.o', 'b.o', 'lib.so'):                      # (made at one time, whatever the file system's resolution)
            os.utime(csrc / name, (2000, 2000))
        return sorted(w for line in lines for w in line.split() if w.endswith('.hip')), any('-shared' in line for line in lines)
    return csrc, made


def _names(result):
    return [os.path.basename(p) for p in result[0]], result[1]


def test_nothing_is_compiled_twice(tree):
    _, made = tree
    assert _names(made()) == (['a.hip', 'b.hip'], True)
    assert _names(made()) == ([], False)
    assert _names(made(force=True)) == (['a.hip', 'b.hip'], True)


@pytest.mark.parametrize('changed,again', [('a.hip', ['a.hip']), ('x.h', ['a.hip', 'b.hip']), ('recipe.py', ['a.hip', 'b.hip'])])
def test_a_change_compiles_what_it_concerns(tree, changed, again):
    """recipe.py stands for build.py itself, which holds the compiler's flags."""
    csrc, made = tree
    made()
    os.utime(csrc / changed, (3000, 3000))
    assert _names(made()) == (again, True)


def test_the_recipe_is_the_file_with_the_flags():
    with open(build.RECIPE) as f:
        assert 'packed-fp32-ops' in f.read()
