"""The build's order and its staleness rule, with a compiler that only writes down what it was asked for."""
import shutil

import pytest

from mojo_llm_lab_b200 import build as B


@pytest.fixture
def made(tmp_path, monkeypatch):
    """build() into an empty folder; the names made so far, and the one whose compiler fails."""
    names, state = [], {"fails": None}
    for attr in ("LIB", "CUBIN", "INTERPOSE", "HARNESS", "TORCH_EXT"):
        monkeypatch.setattr(B, attr, tmp_path / getattr(B, attr).name)
    monkeypatch.setattr(B, "LIBDIR", tmp_path)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")

    def run(cmd, log, verbose):
        out = next(cmd[i + 1] for i, x in enumerate(cmd) if x == "-o")
        name = out.rsplit("/", 1)[-1].replace(".tmp", "")
        if name == state["fails"]:
            raise RuntimeError(f"{cmd[0]} failed")
        open(out, "w").close()
        names.append(name)

    monkeypatch.setattr(B, "_run", run)
    return names, state


C_PARTS = {"libmllb200.so", "libmllb200_interpose.so", "mllb200_harness", "mllb200_compat.cubin"}


def test_the_c_parts_build_without_torch(made, monkeypatch):
    monkeypatch.setattr(B, "_torch_stamp", lambda: None)
    B.build()
    assert set(made[0]) == C_PARTS


def test_the_c_parts_are_made_before_the_extension_can_fail(made):
    made[1]["fails"] = "mllb200_torch.so"
    with pytest.raises(RuntimeError):
        B.build()
    assert set(made[0]) == C_PARTS


def test_the_extension_follows_torch_and_python(made, monkeypatch):
    B.build()
    assert made[0][-1] == "mllb200_torch.so" and B.torch_ext_current()
    made[0].clear()
    B.build()
    assert made[0] == []
    monkeypatch.setattr(B, "_torch_stamp", lambda: "another torch")
    assert not B.torch_ext_current()
    B.build()
    assert made[0] == ["mllb200_torch.so"] and B.torch_ext_current()


def test_a_failing_compiler_is_named(tmp_path):
    with pytest.raises(RuntimeError, match="false failed"):
        B._run([shutil.which("false")], tmp_path / "log", False)
