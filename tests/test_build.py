"""pixelssl_amd.build: the C library does not wait on the autograd nodes, which follow torch's version."""
import os

import pytest


@pytest.fixture
def tools(monkeypatch, tmp_path):
    """compilers that only touch their output"""
    from pixelssl_amd import build as B
    made = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        made.append(os.path.basename(out))
        open(out, "w").write("x")
        return Done()

    monkeypatch.setattr(B, "OBJDIR", str(tmp_path / "obj"))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libpixelhip.so"))
    monkeypatch.setattr(B, "NODE_LIB", str(tmp_path / "_pxlnode.so"))
    monkeypatch.setattr(B, "NODE_STAMP", str(tmp_path / "obj" / "_pxlnode.cmd"), raising=False)
    monkeypatch.setattr(B.subprocess, "run", run)
    return B, made


def test_the_library_is_linked_though_the_nodes_do_not_compile(tools, monkeypatch):
    B, made = tools

    def broken(force):
        raise RuntimeError("no such header")

    monkeypatch.setattr(B, "_build_node", broken)
    with pytest.raises(RuntimeError, match="no such header"):
        B.build(verbose=False)
    assert "libpixelhip.so" in made and os.path.exists(B.LIB)


def test_the_library_alone(tools, monkeypatch):
    B, made = tools
    monkeypatch.setattr(B, "_build_node", lambda force: pytest.fail("not asked for"))
    assert B.build(verbose=False, node=False) == B.LIB and "libpixelhip.so" in made and "_pxlnode.so" not in made


def test_the_nodes_follow_torch(tools, monkeypatch):
    import torch
    B, made = tools
    B.build(verbose=False)
    assert "_pxlnode.so" in made
    made.clear()
    B.build(verbose=False)
    assert made == []
    monkeypatch.setattr(torch, "__version__", "99.0")
    B.build(verbose=False)
    assert made == ["_pxlnode.so"]
