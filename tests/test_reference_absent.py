"""CPU: a missing build of the reference is passed over only where the tree that it
is made from is missing too; with the tree there it is an error."""
import json
import types

import pytest

import bench
import pyoracle
from conftest import reference_absent


@pytest.mark.parametrize("tree", [True, False])
def test_what_counts_as_absent(monkeypatch, tree):
    monkeypatch.setattr(pyoracle, "ref_tree", lambda: tree)
    for path in (pyoracle.LIB_REF, pyoracle.LIB_REF_DEC, pyoracle.LIB_REF_FULL):
        assert reference_absent(FileNotFoundError(path)) is not tree
        assert not reference_absent(RuntimeError(path))
    assert not reference_absent(FileNotFoundError(pyoracle.LIB_REF + ".old"))
    assert not reference_absent(FileNotFoundError(2, "no such file", "oracle/_ref/other"))


def test_the_tree_is_the_makefiles(monkeypatch, tmp_path):
    monkeypatch.setenv("REF", str(tmp_path))
    assert not pyoracle.ref_tree()
    (tmp_path / "tensor_ops.c").write_text("")
    assert pyoracle.ref_tree()


@pytest.mark.parametrize("tree", [True, False])
def test_bench_reference_arm(monkeypatch, capsys, tree):
    def missing(*a):
        raise FileNotFoundError(pyoracle.LIB_REF)
    monkeypatch.setattr(bench, "RefRunner", missing)
    monkeypatch.setattr(pyoracle, "ref_tree", lambda: tree)
    args = types.SimpleNamespace(T=375, blocks=1, steps=1, warmup=3)
    if tree:
        with pytest.raises(FileNotFoundError):
            bench.reference_arm(args, 0, 1)
    else:
        bench.reference_arm(args, 0, 1)
        line = json.loads(capsys.readouterr().out)
        assert line["impl"] == "reference" and "absent" in line["unavailable"]
