"""What the Makefile builds again: a copy of the sources with stand-ins for the built files, asked with `make -q` and `make -n`
(nothing is compiled)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "unet_amd", "csrc")
LIBRARY, BINDING = "../libunetmi.so", "../libunetmi_torch.so"


class Tree:
    def __init__(self, root):
        self.root, self.csrc = root, root / "unet_amd" / "csrc"
        self.csrc.mkdir(parents=True)
        (root / "include").mkdir()
        shutil.copy(os.path.join(ROOT, "include", "unetmi.h"), root / "include")
        for name in os.listdir(CSRC):
            if name == "Makefile" or name.endswith((".hip", ".hpp", ".cpp")):
                shutil.copy(os.path.join(CSRC, name), self.csrc)
        self.kernels = [n for n in os.listdir(self.csrc) if n.endswith(".hip")]
        self.use_torch("torch_a")

    def use_torch(self, name, version="1"):
        """The interpreter that the Makefile asks where torch is answers with this folder."""
        (self.root / name).mkdir(exist_ok=True)
        (self.root / name / "version.py").write_text("__version__ = '{}'\n".format(version))
        (self.root / "python").write_text("#!/bin/sh\necho {}\n".format(self.root / name))
        (self.root / "python").chmod(0o755)

    def make(self, *args):
        return subprocess.run(["make", "-C", str(self.csrc), "PYTHON={}".format(self.root / "python"), *args], capture_output=True, text=True)

    def stale(self, target, *settings):
        answer = self.make("-q", target, *settings)
        assert answer.returncode in (0, 1), answer.stderr
        return answer.returncode == 1

    def compiled(self, *settings):
        """The commands that would compile kernels."""
        return [line for line in self.make("-n", LIBRARY, *settings).stdout.splitlines() if " -c " in line]

    def built(self, *settings):
        """As after a build a while ago: every source older than what is built from it."""
        self.make("-n", *settings)
        for folder, _, names in os.walk(self.root):
            for name in names:
                os.utime(os.path.join(folder, name), (1e9, 1e9))
        for path in [self.csrc / (n[:-4] + ".o") for n in self.kernels] + [self.csrc / BINDING, self.csrc / LIBRARY]:
            path.touch()
            os.utime(path, (1.1e9, 1.1e9) if path.name.endswith(".o") else (1.2e9, 1.2e9))
        return self


@pytest.fixture
def tree(tmp_path):
    return Tree(tmp_path).built()


def test_only_what_changed_is_built_again(tree):
    assert not tree.stale(LIBRARY) and not tree.stale(BINDING)
    (tree.csrc / "seq_conv.hip").touch()
    assert tree.stale(LIBRARY) and not tree.stale(BINDING)
    assert len(tree.compiled()) == 1 and "seq_conv.hip" in tree.compiled()[0]


def test_a_changed_makefile_builds_everything_again(tree):
    (tree.csrc / "Makefile").touch()
    assert len(tree.compiled()) == len(tree.kernels) and tree.stale(BINDING)


def test_other_flags_build_the_kernels_again_and_never_with_packed_fp32(tree):
    flags = "CXXFLAGS=-O1 --offload-arch=gfx950"
    for settings, level in (((flags,), " -O1 "), ((), " -O3 ")):
        commands = tree.compiled(*settings)
        assert len(commands) == len(tree.kernels)
        assert all(level in c and "-Xclang -target-feature -Xclang -packed-fp32-ops" in c for c in commands)
        assert not tree.stale(BINDING, *settings)
        tree.built(*settings)
        assert not tree.compiled(*settings)


def test_another_torch_builds_the_binding_again(tree):
    for name, version in (("torch_b", "1"), ("torch_b", "2")):
        tree.use_torch(name, version)
        assert tree.stale(BINDING) and not tree.stale(LIBRARY)
        assert name in tree.make("-n", BINDING).stdout
        tree.built()
        assert not tree.stale(BINDING)
