"""What the build writes appears whole: processes that start together may each
build the torch binding on its first use."""

import os
from types import SimpleNamespace

import pytest

from private_genomic_dnagpt_b200 import build


@pytest.mark.parametrize("fails", [False, True])
def test_the_binding_appears_whole_or_not_at_all(monkeypatch, tmp_path, fails):
    pytest.importorskip("torch")
    out = str(tmp_path / "_draft.so")
    monkeypatch.setattr(build, "BINDING", out)

    def compiler(cmd, **kw):
        target = cmd[cmd.index("-o") + 1]
        with open(target, "w") as f:
            f.write("half")
            f.flush()
            # another process looks now
            assert not os.path.exists(out)
            f.write(" and half")
        return SimpleNamespace(returncode=int(fails), stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    if fails:
        with pytest.raises(RuntimeError, match="g.. failed"):
            build.build_binding()
        assert os.listdir(tmp_path) == []
    else:
        assert build.build_binding() == out
        assert os.listdir(tmp_path) == ["_draft.so"] and open(out).read() == "half and half"
