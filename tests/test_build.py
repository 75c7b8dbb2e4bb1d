"""What zeno_b200/build.py leaves behind (no compiler runs: the commands are recorded and their outputs touched)."""
import pytest

from zeno_b200 import build as zbuild


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """An empty tree with a PyTorch; ``commands``: what was run; ``broken``: the files that do not compile."""
    class Tree:
        commands, broken = [], set()
        torch = tmp_path / "torch"
        lib, binding, copy = (tmp_path / n for n in ("lib/libzeno.so", "lib/zeno_torch.so", "zig-out/lib/libzeno.so"))

        def build(self, **kw):
            del self.commands[:]
            return zbuild.build(**kw)

    def runner(verbose):
        def run(cmd):
            Tree.commands.append(cmd)
            if any(str(c).endswith(b) for c in cmd for b in Tree.broken):
                raise RuntimeError("build failed: " + " ".join(cmd))
            out = cmd[cmd.index("-o") + 1]
            open(out, "w").write("built")
        return run
    Tree.commands, Tree.broken = [], set()
    for name, value in (("OUT_DIR", tmp_path / "lib"), ("LIB", Tree.lib), ("BINDING", Tree.binding), ("OBJ_DIR", tmp_path / "_build"),
                        ("BINDING_STAMP", tmp_path / "lib" / "zeno_torch.txt"), ("ZIG_OUT_LIB", Tree.copy), ("_runner", runner)):
        monkeypatch.setattr(zbuild, name, value, raising=False)
    (Tree.torch / "lib").mkdir(parents=True)
    (Tree.torch / "lib" / "libtorch_cuda.so").write_text("")
    (Tree.torch / "__init__.py").write_text("")
    (Tree.torch / "version.py").write_text("__version__ = '1'")
    headers = tmp_path / "include"
    headers.mkdir()
    (headers / "Python.h").write_text("")
    Tree.headers = headers

    class Spec:
        origin = str(Tree.torch / "__init__.py")
    monkeypatch.setattr(zbuild.importlib.util, "find_spec", lambda name: Spec if Tree.torch else None)
    monkeypatch.setattr(zbuild.sysconfig, "get_paths", lambda: {"include": str(headers)})
    return Tree()


def test_all_of_it_once(tree):
    assert tree.build() == tree.lib
    assert tree.lib.exists() and tree.copy.exists() and tree.binding.exists()
    tree.build()
    assert not tree.commands


def test_the_library_and_its_copy_do_not_wait_for_the_pytorch_functions(tree):
    tree.broken.add("torch_binding.cpp")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="torch_binding"):
            tree.build()
        assert tree.lib.exists() and tree.copy.exists() and not tree.binding.exists()
    tree.broken.clear()
    tree.build()
    assert tree.binding.exists() and len(tree.commands) == 2


def test_a_missing_or_older_copy_is_made(tree):
    tree.build()
    tree.copy.unlink()
    tree.build()
    assert tree.copy.read_text() == "built" and not tree.commands


@pytest.mark.parametrize("without", ["PyTorch", "CUDA", "headers"])
def test_without_a_pytorch_to_build_against(tree, without):
    if without == "PyTorch":
        type(tree).torch = None
    elif without == "CUDA":
        (tree.torch / "lib" / "libtorch_cuda.so").unlink()
    else:
        (tree.headers / "Python.h").unlink()
    tree.build()
    assert tree.lib.exists() and tree.copy.exists() and not tree.binding.exists()


def test_another_pytorch_is_built_against(tree):
    tree.build()
    (tree.torch / "version.py").write_text("__version__ = '2'")
    tree.build()
    assert len(tree.commands) == 2 and all("zeno_torch" in " ".join(c) or "torch_binding" in " ".join(c) for c in tree.commands)
    tree.build()
    assert not tree.commands
