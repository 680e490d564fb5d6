"""CPU: what makes build.sh compile an object again -- its sources, and build.sh itself, which holds the compiler's flags (one of them decides whether results are right).
The compilers are stand-ins that only make the output file."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_flags_are_a_dependency_of_every_object(tmp_path):
    csrc = tmp_path / 'merlot_amd' / 'csrc'
    shutil.copytree(os.path.join(ROOT, 'include'), tmp_path / 'include')
    shutil.copytree(os.path.join(ROOT, 'merlot_amd', 'csrc'), csrc, ignore=shutil.ignore_patterns('build', 'build_exp', '*.o', '*.so'))
    bin_ = tmp_path / 'bin'
    bin_.mkdir()
    for name in ('hipcc', 'g++'):                             # each call leaves its arguments behind
        f = bin_ / name
        f.write_text('#!/bin/bash\necho "$0 $*" >> %s/calls\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n' % tmp_path)
        f.chmod(0o755)
    # every file older than the objects to come
    for d, _, files in os.walk(tmp_path):
        for f in files:
            os.utime(os.path.join(d, f), (1e9, 1e9))

    def build(**env):
        (tmp_path / 'calls').write_text('')
        subprocess.run(['bash', str(csrc / 'build.sh')], check=True, capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, HIPCC=str(bin_ / 'hipcc'), PATH=f'{bin_}:' + os.environ['PATH'], **env))
        man = (csrc / 'build' / 'BUILD_MANIFEST').read_text().split()
        return dict(zip(man[1::2], man[0::2])), (tmp_path / 'calls').read_text()
    man, calls = build()
    n = len(man)
    assert n >= 17 and set(man.values()) == {'compiled'} and 'probe.hip' in calls
    assert all('-packed-fp32-ops' in c for c in calls.splitlines() if '.hip ' in c)      # (no object without the flag that keeps the packed instructions out)
    man, calls = build()
    assert set(man.values()) == {'reused'} and 'probe.hip' not in calls
    os.utime(csrc / 'clip.hip')
    man, _ = build()
    assert [k for k, v in man.items() if v == 'compiled'] == ['clip.o']
    os.utime(csrc / 'build.sh', (4e9, 4e9))                    # newer than every object
    man, calls = build()
    assert set(man.values()) == {'compiled'} and 'probe.hip' in calls
    os.utime(csrc / 'build.sh', (1e9, 1e9))
    man, _ = build()
    assert set(man.values()) == {'reused'}
    man, calls = build(MERLOT_BUILD_ALL='1')
    assert len(man) == n and set(man.values()) == {'compiled'} and 'probe.hip' in calls


def test_the_entry_point_compiles_everything(monkeypatch):
    import __graft_entry__ as entry
    seen = {}
    monkeypatch.setattr(entry.subprocess, 'check_call', lambda cmd, env: seen.update(cmd=cmd, env=env))
    entry.build()
    assert seen['cmd'][-1].endswith('build.sh') and seen['env']['MERLOT_BUILD_ALL'] == '1'
