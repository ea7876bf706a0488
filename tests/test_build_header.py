"""The torch module is compiled against the C header: a header that changed after it was built makes it stale. (The structs that it passes are declared there.)"""
import os
import time

from test_build import B, tree  # noqa: F401 (a fixture)


def test_the_module_follows_the_header(tree, tmp_path, monkeypatch):  # noqa: F811
    include = tmp_path / "include"
    include.mkdir()
    (include / "xnq.h").write_text("// nothing\n")
    here = tmp_path / "package"
    here.mkdir()
    monkeypatch.setattr(B, "HERE", str(here))
    B.build_torch_module()
    assert not B.torch_module_is_stale()
    later = time.time() + 10
    os.utime(include / "xnq.h", (later, later))
    assert B.torch_module_is_stale()
    B.build_torch_module()
    assert len(tree) == 2
