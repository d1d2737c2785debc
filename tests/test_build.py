"""The in-tree build keeps an object only while its command, compiler, source and headers are what it was made from.
The compilers are stand-ins that write what they were asked for; the sources are a copy of the tree's."""
import os
import shutil

import pytest

from mx_rcnn_amd.csrc import build as B


@pytest.fixture
def fake(tmp_path, monkeypatch):
    here = tmp_path / 'csrc'
    shutil.copytree(B.HERE, str(here), ignore=shutil.ignore_patterns('_build', '__pycache__'))
    monkeypatch.setattr(B, 'HERE', str(here))
    monkeypatch.setattr(B, 'BUILD', str(here / '_build'))
    monkeypatch.setenv('MXR_EXT_OUT', str(tmp_path / 'out.so'))
    monkeypatch.delenv('MXR_SYNC_DEBUG', raising=False)

    class Fake(object):
        version, fails, ran = 'one', None, []

        def run(self, cmd):
            if cmd[1] == '--version':
                return self.version
            out = cmd[cmd.index('-o') + 1]
            if self.fails and self.fails in os.path.basename(out):
                raise RuntimeError('build step failed')
            self.ran.append(os.path.basename(out))
            with open(out, 'w') as f:
                f.write('%d' % len(self.ran))
            return ''

        def build(self, **kw):
            self.ran = []
            B.build(jobs=1, **kw)
            return set(self.ran)

        here = str(tmp_path / 'csrc')
    f = Fake()
    monkeypatch.setattr(B, '_run', f.run)
    return f


def test_kept_and_rebuilt(fake, monkeypatch):
    first = fake.build()
    hips = {n + '.o' for n in os.listdir(os.path.join(fake.here, 'hip')) if n.endswith('.hip')}
    assert first == hips | {'bindings.o', 'out.so'}
    assert fake.build() == set()
    # a newer date alone changes nothing, an older one with other text does
    src = os.path.join(fake.here, 'hip', 'sgd.hip')
    os.utime(src)
    assert fake.build() == set()
    with open(src, 'a') as f:
        f.write('// more\n')
    os.utime(src, (1, 1))
    assert fake.build() == {'sgd.hip.o', 'out.so'}
    # a header: what includes it
    with open(os.path.join(fake.here, 'hip', 'tile_nt.h'), 'a') as f:
        f.write('// more\n')
    assert fake.build() == {'newton_schulz.hip.o', 'int8_gemm.hip.o', 'out.so'}
    # flags and compilers
    monkeypatch.setenv('MXR_SYNC_DEBUG', '1')
    assert fake.build() == hips | {'out.so'}
    assert fake.build(debug=True) == first
    assert fake.build(debug=True) == set()
    fake.version = 'two'
    assert fake.build(debug=True) == first
    # the library: gone, or another file in its place
    out = os.environ['MXR_EXT_OUT']
    os.remove(out)
    assert fake.build(debug=True) == {'out.so'}
    with open(out, 'a') as f:
        f.write('x')
    assert fake.build(debug=True) == {'out.so'}
    assert fake.build(debug=True, force=True) == first


def test_failed_step_is_done_again(fake):
    fake.build()
    src = os.path.join(fake.here, 'hip', 'sgd.hip')
    with open(src) as f:
        text = f.read()
    with open(src, 'a') as f:
        f.write('broken')
    fake.fails = 'sgd'
    with pytest.raises(RuntimeError):
        fake.build()
    with open(src, 'w') as f:
        f.write(text)  # as it was: the object may be half written all the same
    fake.fails = None
    assert fake.build() == {'sgd.hip.o', 'out.so'}
