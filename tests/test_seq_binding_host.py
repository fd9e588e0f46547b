"""The sequence operators without their host binding (CPU)."""
import subprocess

import pytest
import torch

from hard_resets_compose_b200 import _lib, embed


@pytest.mark.parametrize("error", (RuntimeError("g++ not found"), subprocess.CalledProcessError(1, ["g++"]),
                                   OSError("read-only file system")))
def test_without_a_compiler(monkeypatch, tmp_path, error):
    """Neither built nor there: a warning, and the Python functions take the calls."""
    def build_binding(*args, **kw):
        raise error
    monkeypatch.setattr(_lib._build, "build_binding", build_binding)
    monkeypatch.setattr(_lib._build, "binding_path", lambda: str(tmp_path / "none.so"))
    monkeypatch.setattr(_lib, "_fast", None)
    with pytest.warns(RuntimeWarning, match="host binding"):
        binding = _lib.fast()
    assert binding.embedding(1, 2, 3) is None and _lib.fast() is binding
    with pytest.raises(RuntimeError, match="CUDA"):  # the Python function's own refusal
        embed.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(4, 2))


def test_a_binding_that_does_not_load(monkeypatch, tmp_path):
    bad = tmp_path / "lifb_seq.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(_lib._build, "build_binding", lambda *a, **k: str(bad))
    monkeypatch.setattr(_lib, "_fast", None)
    with pytest.warns(RuntimeWarning, match="host binding"):
        assert _lib.fast().norm_gate() is None
