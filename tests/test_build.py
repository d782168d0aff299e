"""The build's order: the C library does not wait for what only the autograd
nodes need."""
import os

import pytest


@pytest.mark.parametrize("missing", ["compiler", "torch's headers", "link"])
def test_the_library_is_linked_without_the_nodes(monkeypatch, tmp_path, missing):
    from concord_amd import build as B
    monkeypatch.setattr(B, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libconcord_amd.so"))
    monkeypatch.setattr(B, "OPS", str(tmp_path / "concord_torch_ops.so"))

    def run(cmd):
        if cmd[0] == B.CXX and (missing == "compiler" or missing == "link" and "-shared" in cmd):
            raise RuntimeError("command failed: g++")
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return ""

    def no_headers():
        raise RuntimeError("no headers")
    monkeypatch.setattr(B, "_run", run)
    if missing == "torch's headers":
        monkeypatch.setattr(B, "_ops_flags", no_headers)
    with pytest.raises(RuntimeError):   # and the failure is not hidden
        B.build()
    assert os.path.exists(B.LIB) and not os.path.exists(B.OPS)


def test_both_are_built(monkeypatch, tmp_path):
    from concord_amd import build as B
    monkeypatch.setattr(B, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libconcord_amd.so"))
    monkeypatch.setattr(B, "OPS", str(tmp_path / "concord_torch_ops.so"))
    order = []

    def run(cmd):
        out = cmd[cmd.index("-o") + 1]
        order.append(os.path.basename(out))
        with open(out, "w"):
            pass
        return ""
    monkeypatch.setattr(B, "_run", run)
    assert B.build() == B.LIB
    assert sorted(os.listdir(tmp_path)) == ["concord_torch_ops.so", "libconcord_amd.so"]
    # (the nodes' module is linked against the library)
    assert order.index("libconcord_amd.so.tmp") < order.index("concord_torch_ops.so.tmp")


def test_a_kernel_that_does_not_compile_links_nothing(monkeypatch, tmp_path):
    from concord_amd import build as B
    monkeypatch.setattr(B, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libconcord_amd.so"))
    monkeypatch.setattr(B, "OPS", str(tmp_path / "concord_torch_ops.so"))

    def run(cmd):
        if any(c.endswith("attention.hip") for c in cmd):
            raise RuntimeError("command failed: hipcc")
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return ""
    monkeypatch.setattr(B, "_run", run)
    with pytest.raises(RuntimeError, match="hipcc"):
        B.build()
    assert not os.path.exists(B.LIB) and not os.path.exists(B.OPS)
