"""The C++ host module is that of the torch that is installed."""
import pytest

from torchft_b200 import _build
from torchft_b200.ops import _native as N


def test_a_module_of_another_torch_is_not_loaded(tmp_path, monkeypatch):
    mine = _build.host_mod()
    assert mine == _build.build_host() and mine.exists()
    other = tmp_path / "torch"
    other.mkdir()
    (other / "version.py").write_text((_build._torch_dir() / "version.py").read_text() + "\n# built again\n")
    monkeypatch.setattr(_build, "_torch_dir", lambda: other)
    assert _build.host_mod() != mine
    monkeypatch.setattr(N, "_host", None)
    monkeypatch.setenv("FTB200_NO_AUTOBUILD", "1")
    with pytest.raises(N.KernelError, match="is missing"):
        N.host()


def test_the_module_is_bound_once():
    assert N.host() is N.host()
    assert N.host().__file__ == str(_build.host_mod())
